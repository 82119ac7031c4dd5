// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = y[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T,   a = ids[t]   (a = -1: out[t] = y[t])
//
// with A [adapters, rank, K], B [adapters, N, rank] bf16 and y the projection's own output (bf16,
// or the LM head's fp32 logits). One launch, no workspace: a cluster of CTAs takes a tile of rows and
// a range of the N outputs. First u = x . A^T: the cluster's CTAs split K, their warps split it again,
// and the partial sums (fp32) are added in a fixed order through distributed shared memory. Then each
// CTA adds u . B^T to its share of the outputs. A tile of several rows goes through the adapters that
// its rows name, one after another; rows of other adapters ride along in the products and are left
// out of the results. Ids may come in any order: where they come mixed, tiles gather the rows of one
// adapter. A decode batch goes one row a tile, without the tensor cores (adapter_row_kernel).
//
// The products are 8 to 128 wide, far too little arithmetic per byte to need tcgen05's staging through
// shared and tensor memory (rank 64: 36 FLOP per byte of x, y and out): mma.sync takes its operands from
// registers, straight from 16-byte global loads. For that the K order inside a step is permuted
// alike in both operands: a lane's consecutive elements fill its places of the fragments. What bounds
// it is the chain of a tile's phases, 5 to 15 us of it, and beyond that mma.sync itself (0.4 a cycle an
// SM): 2,048 rows of 768 -> 3,072, rank 64, 26 us, 0.18 of what x, y and out cost at the copy rate.
//
// u is carried into the second product as a sum of bf16 numbers: two of them (off by 2^-17 of u at most)
// for bf16 outputs, whose own rounding is 2^-8, and three, which hold all of an fp32 number's 24 bits, for
// an adapted head's fp32 logits (with two these were 2e-6 off, with three 1e-7).
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxRank = 128, kMaxCluster = 8;
constexpr int kMaxSort = 1024;         // adapters up to which rows are gathered by adapter
constexpr int kWindow = 4096;          // rows among which they are

struct AdapterArgs {
    const uint16_t *x;
    int T, K, N;
    const uint16_t *a, *b;
    const float *scale;
    int adapters, rank;
    const int32_t *ids;
    const void *y;
    void *out;
    int rows, splits;                  // rows per tile, ranges of N per tile
    int sort;                          // gather rows by adapter where they come mixed
    int vec;                           // rows of y and out start at 16-byte boundaries
};

MOE_D void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

MOE_D uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// what a bf16 drops of v; nothing of what is not finite
MOE_D float below_bf16(float v) {
    const float r = bf16r(v);
    return fabsf(r) < INFINITY ? v - r : 0.f;
}

// kMT: row fragments (16 rows) a tile; kNT: fragments of 8 rank rows the warps have registers for
template <int kMT, int kNT, int kParts>
struct Smem {
    static constexpr int kRows = 16 * kMT, kWK = kWarps / kMT;       // warps along K per row fragment
    static constexpr int kR = 8 * kNT, kSteps = (kR + 15) / 16;
    static constexpr int kF = kNT == 2 ? 8 : 4;  // output fragments of 8 a warp takes at a time
    float part[kWK][kRows][kR];        // the warps' sums over their K steps
    float u[kRows][kR];                // the CTA's sums, read by the cluster
    uint4 frag[kParts][kMT][kSteps][32];         // scale * u as fragments: high to low parts
    int row[kRows], id[kRows];         // the tile's rows and their adapters
    int kind[kRows];                   // the different ones among them
    unsigned member[kRows];            // which rows are of that kind
    int kinds, sums[kWarps];
    // gathering: the window's rows' adapters, and the places of each adapter's rows
    uint16_t bin[kWindow], near[kWindow];
    int start[kMaxSort + 2], next[kMaxSort + 1];
};

// 8 consecutive outputs as they lie in memory (left of them are inside the row)
template <bool kFp32>
struct Out8 {
    uint32_t w[kFp32 ? 8 : 4];
    MOE_D float get(int i) const {
        return kFp32 ? __uint_as_float(w[i]) : __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
    MOE_D void set2(int i, float a, float b) {       // outputs i (even) and i + 1
        if (kFp32) {
            w[i] = __float_as_uint(a);
            w[i + 1] = __float_as_uint(b);
        } else {
            w[i >> 1] = pack_bf16(a, b);
        }
    }
    // whole: all 8 lie inside a row that starts at a 16-byte boundary
    MOE_D void load(const void *y, size_t at, bool whole, int left) {
        constexpr int kW = kFp32 ? 8 : 4;
        if (whole) {
            const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(y) + at * (kFp32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < kW / 4; ++i) {
                const uint4 q = p[i];
                w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
            }
        } else if (kFp32) {
#pragma unroll
            for (int i = 0; i < kW; ++i) w[i] = i < left ? static_cast<const uint32_t *>(y)[at + i] : 0u;
        } else {
            const uint16_t *p = static_cast<const uint16_t *>(y) + at;
#pragma unroll
            for (int i = 0; i < kW; ++i)
                w[i] = (2 * i < left ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)p[2 * i + 1] << 16 : 0u);
        }
    }
    MOE_D void store(void *out, size_t at, bool whole, int left) const {
        constexpr int kW = kFp32 ? 8 : 4;
        if (whole) {
            uint4 *p = reinterpret_cast<uint4 *>(static_cast<char *>(out) + at * (kFp32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < kW / 4; ++i) p[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else if (kFp32) {
#pragma unroll
            for (int i = 0; i < kW; ++i)
                if (i < left) static_cast<uint32_t *>(out)[at + i] = w[i];
        } else {
            uint16_t *p = static_cast<uint16_t *>(out) + at;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
};

// The rows of a tile, in sh.row / sh.id. Rows come in the order given when that keeps those of one
// adapter together (a prompt's rows, one adapter for all); otherwise the rows of the tile's window are
// taken in the order of their adapters (rows of one adapter in order, rows without one last): the tile
// then holds few adapters, and each is read by few tiles.
template <class S>
MOE_D int tile_rows(S &sh, const AdapterArgs &p, int tile, bool report) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = kWindow / p.rows, w0 = tile / per * per * p.rows, wn = min(p.T - w0, per * p.rows);
    const int at = tile * p.rows - w0, rows = min(p.rows, wn - at);
    const int32_t *ids = p.ids + w0;
    bool mixed = false;
    if (p.sort) {
        int runs = 0;
        constexpr int kB = 8;                    // ids a thread has in flight
        for (int t0 = tid; t0 < wn; t0 += kB * kThreads) {
            int id[kB], before[kB];
#pragma unroll
            for (int i = 0; i < kB; ++i) {
                const int t = t0 + i * kThreads;
                id[i] = t < wn ? __ldg(ids + t) : 0;
                before[i] = t < wn && t > 0 ? __ldg(ids + t - 1) : ~id[i];
            }
#pragma unroll
            for (int i = 0; i < kB; ++i) {
                const int t = t0 + i * kThreads;
                if (t >= wn) break;
                runs += id[i] != before[i] ? 1 : 0;
                const bool in = id[i] >= 0 && id[i] < p.adapters;
                if (!in && id[i] != -1 && report) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
                sh.bin[t] = (uint16_t)(in ? id[i] : p.adapters);
            }
        }
        for (int i = tid; i <= p.adapters; i += kThreads) sh.next[i] = 0;
        runs = __reduce_add_sync(0xffffffffu, runs);
        if (lane == 0) sh.sums[warp] = runs;
        __syncthreads();
        runs = 0;
        for (int w = 0; w < kWarps; ++w) runs += sh.sums[w];
        mixed = runs * p.rows > 2 * wn;          // runs shorter than half a tile
    }
    if (tid < S::kRows) {
        int id = -1;
        if (tid < rows) {
            id = p.sort ? (int)sh.bin[at + tid] : ids[at + tid];
            if (p.sort && id == p.adapters) id = -1;
            if (id < -1 || id >= p.adapters) {
                if (report) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
                id = -1;
            }
        }
        sh.row[tid] = w0 + at + min(tid, rows - 1);
        sh.id[tid] = id;
    }
    if (!mixed) {
        __syncthreads();
        return rows;
    }
    for (int t = tid; t < wn; t += kThreads) atomicAdd(&sh.next[sh.bin[t]], 1);
    __syncthreads();
    if (warp == 0) {
        int before = 0;                          // places: an exclusive scan of the counts
        for (int i0 = 0; i0 <= p.adapters; i0 += 32) {
            const int i = i0 + lane, c = i <= p.adapters ? sh.next[i] : 0;
            int sum = c;
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, sum, off);
                if (lane >= off) sum += o;
            }
            if (i <= p.adapters) sh.start[i] = sh.next[i] = before + sum - c;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) sh.start[p.adapters + 1] = before;
    }
    __syncthreads();
    // the rows of the adapters that reach the tile: every warp lists those of its share of the window, in order
    constexpr int kShare = kWindow / kWarps;
    const int each = ((wn + kWarps - 1) / kWarps + 31) & ~31, t1 = min((warp + 1) * each, wn);
    int found = 0;
    for (int t0 = warp * each; t0 < t1; t0 += 32) {
        const int t = t0 + lane, b = t < t1 ? sh.bin[t] : -1;
        const bool near = b >= 0 && sh.start[b] < at + rows && sh.start[b + 1] > at;
        const unsigned who = __ballot_sync(0xffffffffu, near);
        if (near) sh.near[warp * kShare + found + __popc(who & ((1u << lane) - 1u))] = (uint16_t)t;
        found += __popc(who);
    }
    if (lane == 0) sh.sums[warp] = found;
    __syncthreads();
    if (warp == 0) {                             // their places, in row order
        for (int w = 0; w < kWarps; ++w) {
            const int n = sh.sums[w];
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int t = i0 + lane < n ? sh.near[w * kShare + i0 + lane] : -1, b = t >= 0 ? sh.bin[t] : -1;
                unsigned todo = __ballot_sync(0xffffffffu, t >= 0);
                while (todo) {
                    const int k = __shfl_sync(0xffffffffu, b, __ffs(todo) - 1);
                    const unsigned who = __ballot_sync(0xffffffffu, b == k);
                    todo &= ~who;
                    const int first = sh.next[k] - at, place = first + __popc(who & ((1u << lane) - 1u));
                    if (b == k && place >= 0 && place < rows) {
                        sh.row[place] = w0 + t;
                        sh.id[place] = b < p.adapters ? b : -1;
                    }
                    __syncwarp();
                    if (lane == 0) sh.next[k] = first + at + __popc(who);
                    __syncwarp();
                }
            }
        }
    }
    __syncthreads();
    return rows;
}

// two CTAs an SM where the registers allow it: the kernel is a chain of short dependent phases
template <int kMT, int kNT, bool kFp32>
__global__ void __launch_bounds__(kThreads, kNT <= 8 ? 2 : 1) adapter_kernel(AdapterArgs p) {
    constexpr int kParts = kFp32 ? 3 : 2;
    using S = Smem<kMT, kNT, kParts>;
    extern __shared__ __align__(16) unsigned char smem[];
    S &sh = *reinterpret_cast<S *>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int unit = blockIdx.x / ctas, tile = unit / p.splits, split = unit % p.splits;
    const int rows = tile_rows(sh, p, tile, rank == 0 && split == 0);

    // ---- the adapters of the tile, in the order of their first rows
    if (warp == 0) {
        int id = lane < S::kRows ? sh.id[lane] : -1, n = 0;
        unsigned todo = __ballot_sync(0xffffffffu, id >= 0);
        while (todo) {
            const int k = __shfl_sync(0xffffffffu, id, __ffs(todo) - 1);
            const unsigned who = __ballot_sync(0xffffffffu, id == k);
            todo &= ~who;
            if (lane == 0) {
                sh.kind[n] = k;
                sh.member[n] = who;
            }
            ++n;
        }
        if (lane == 0) sh.kinds = n;
    }
    __syncthreads();
    const int kinds = sh.kinds;

    // ---- u = x . A^T: this CTA's part of K, this warp's 32-element steps of it
    const int nt = p.rank / 8;
    if (kinds > 0) {
        const int mt = warp % kMT, wk = warp / kMT;
        const int steps = (p.K + 31) / 32, per = (steps + ctas - 1) / ctas;
        const int s1 = min((rank + 1) * per, steps);
        const int ra = 16 * mt + g, rb = ra + 8;
        const uint16_t *xa = p.x + (size_t)sh.row[ra] * p.K + 8 * q, *xb = p.x + (size_t)sh.row[rb] * p.K + 8 * q;
        const bool oka = ra < rows, okb = rb < rows;
        for (int d = 0; d < kinds; ++d) {
            if (!((sh.member[d] >> (16 * mt)) & 0xffffu)) continue;               // none of this warp's rows
            const uint16_t *ar = p.a + ((size_t)sh.kind[d] * p.rank + g) * p.K + 8 * q;
            float acc[kNT][4] = {};
#pragma unroll (kNT <= 4 ? 4 : kNT <= 8 ? 2 : 1)
            for (int s = rank * per + wk; s < s1; s += S::kWK) {
                const bool in = 32 * s + 8 * q < p.K;
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                const uint4 va = in && oka ? __ldg(reinterpret_cast<const uint4 *>(xa + 32 * s)) : zero;
                const uint4 vb = in && okb ? __ldg(reinterpret_cast<const uint4 *>(xb + 32 * s)) : zero;
                const uint16_t *as = ar + 32 * s;
                uint4 w[kNT];
#pragma unroll
                for (int j = 0; j < kNT; ++j) {
                    w[j] = in && j < nt ? __ldg(reinterpret_cast<const uint4 *>(as)) : zero;
                    as += 8 * p.K;
                }
#pragma unroll
                for (int j = 0; j < kNT; ++j) mma16816(acc[j], va.x, vb.x, va.y, vb.y, w[j].x, w[j].y);
#pragma unroll
                for (int j = 0; j < kNT; ++j) mma16816(acc[j], va.z, vb.z, va.w, vb.w, w[j].z, w[j].w);
            }
            const bool mine = sh.id[ra] == sh.kind[d], mineb = sh.id[rb] == sh.kind[d];
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
                if (mine) *reinterpret_cast<float2 *>(&sh.part[wk][ra][8 * j + 2 * q]) = make_float2(acc[j][0], acc[j][1]);
                if (mineb) *reinterpret_cast<float2 *>(&sh.part[wk][rb][8 * j + 2 * q]) = make_float2(acc[j][2], acc[j][3]);
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < S::kRows * S::kR; i += kThreads) {
        const int r = i / S::kR, c = i % S::kR;
        float s = 0.f;
        if (sh.id[r] >= 0 && c < p.rank) {       // (behind the rank: 0 times what x holds, an infinity too)
#pragma unroll
            for (int w = 0; w < S::kWK; ++w) s += sh.part[w][r][c];
        }
        sh.u[r][c] = s;
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();
    // ---- the cluster's sums, scaled, as fragments
    for (int i = tid; i < kMT * S::kSteps * 32; i += kThreads) {
        const int l = i & 31, s = (i >> 5) % S::kSteps, m = (i >> 5) / S::kSteps;
        const int c = 16 * s + 4 * (l & 3);
        uint32_t f[kParts][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * m + (l >> 2) + 8 * h;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < S::kR && sh.id[r] >= 0) {
                float4 o[kMaxCluster];
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k)
                    o[k] = k < ctas ? *reinterpret_cast<const float4 *>(cluster.map_shared_rank(&sh.u[r][c], k))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    v.x += o[k].x; v.y += o[k].y; v.z += o[k].z; v.w += o[k].w;
                }
                const float scale = __ldg(p.scale + sh.id[r]);
                v.x *= scale; v.y *= scale; v.z *= scale; v.w *= scale;
            }
#pragma unroll
            for (int q3 = 0; q3 < kParts; ++q3) {
                f[q3][h] = pack_bf16(v.x, v.y);
                f[q3][2 + h] = pack_bf16(v.z, v.w);
                v = make_float4(below_bf16(v.x), below_bf16(v.y), below_bf16(v.z), below_bf16(v.w));
            }
        }
#pragma unroll
        for (int q3 = 0; q3 < kParts; ++q3) sh.frag[q3][m][s][l] = make_uint4(f[q3][0], f[q3][1], f[q3][2], f[q3][3]);
    }
    __syncthreads();
    if (ctas > 1) cluster.barrier_arrive();      // this CTA has read the others' u (waited for at the end)

    // ---- out = y + u . B^T, kCols outputs a warp at a time: fragment f, place (q, e) is output
    // n0 + 32 (f / 4) + 8 q + 2 (f % 4) + e, so that a lane ends with runs of 8 consecutive ones
    constexpr int kF = S::kF, kCols = 8 * kF, kChunk = S::kSteps < 4 ? S::kSteps : 4;
    const int groups = (p.N + kCols - 1) / kCols, shares = p.splits * ctas;
    const int share = split * ctas + rank;
    const int gper = (groups + shares - 1) / shares, g0 = min(share * gper, groups), g1 = min(g0 + gper, groups);
    const int steps = (p.rank + 15) / 16;
    size_t at[kMT][2];                           // the lane's rows in y and out
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) at[m][h] = (size_t)sh.row[16 * m + g + 8 * h] * p.N + 8 * q;
    for (int gr = g0 + warp; gr < g1; gr += kWarps) {
        const int n0 = gr * kCols, left = p.N - n0 - 8 * q;
        const bool inner = n0 + kCols <= p.N, whole = inner && p.vec;              // (warp-uniform)
        // fragment column g of fragment f: output n0 + 32 (f / 4) + 8 (g / 2) + 2 (f % 4) + g % 2
        const int nb = n0 + 8 * (g >> 1) + (g & 1);
        for (int d = 0; d < kinds; ++d) {
            const unsigned member = sh.member[d] >> g;
            Out8<kFp32> v[kMT][2][kF / 4];
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < kF / 4; ++c)
                        if (member & (1u << (16 * m + 8 * h)))
                            v[m][h][c].load(p.y, at[m][h] + n0 + 32 * c, whole, left - 32 * c);
            float sum[kMT][kF][4] = {};
            const uint16_t *br = p.b + ((size_t)sh.kind[d] * p.N + nb) * p.rank + 4 * q;
#pragma unroll
            for (int s0 = 0; s0 < S::kSteps; s0 += kChunk) {
                if (s0 >= steps) break;
                uint2 w[kChunk][kF];
#pragma unroll
                for (int f = 0; f < kF; ++f) {
                    const int n = 32 * (f >> 2) + 2 * (f & 3);
                    const uint16_t *bf = br + n * p.rank + 16 * s0;
                    const bool in = inner || nb + n < p.N;
#pragma unroll
                    for (int s = 0; s < kChunk; ++s)
                        w[s][f] = in && 16 * (s0 + s) + 4 * q < p.rank ? __ldg(reinterpret_cast<const uint2 *>(bf + 16 * s))
                                                                       : make_uint2(0u, 0u);
                }
#pragma unroll
                for (int s = 0; s < kChunk; ++s) {
                    if (s0 + s >= steps) break;
#pragma unroll
                    for (int m = 0; m < kMT; ++m) {
                        if (kMT > 1 && !(sh.member[d] & (0xffffu << (16 * m)))) continue;
#pragma unroll
                        for (int h = 0; h < kParts; ++h) {
                            const uint4 u = sh.frag[h][m][s0 + s][lane];
#pragma unroll
                            for (int f = 0; f < kF; ++f) mma16816(sum[m][f], u.x, u.y, u.z, u.w, w[s][f].x, w[s][f].y);
                        }
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < kF / 4; ++c) {
                        if (!(member & (1u << (16 * m + 8 * h)))) continue;
                        Out8<kFp32> &o = v[m][h][c];
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            o.set2(2 * f, o.get(2 * f) + sum[m][4 * c + f][2 * h],
                                   o.get(2 * f + 1) + sum[m][4 * c + f][2 * h + 1]);
                        o.store(p.out, at[m][h] + n0 + 32 * c, whole, left - 32 * c);
                    }
        }
    }
    if (p.out != p.y) {                          // rows without an adapter keep their bits
#pragma unroll
        for (int i = 0; i < 2 * kMT; ++i) {
            const int r = 8 * i + g;
            if (r >= rows || sh.id[r] >= 0) continue;
            for (int gr = g0 + warp; gr < g1; gr += kWarps) {
                const int n0 = gr * kCols, left = p.N - n0 - 8 * q;
                const bool whole = n0 + kCols <= p.N && p.vec;
#pragma unroll
                for (int c = 0; c < kF / 4; ++c) {
                    Out8<kFp32> v;
                    v.load(p.y, at[i / 2][i % 2] + n0 + 32 * c, whole, left - 32 * c);
                    v.store(p.out, at[i / 2][i % 2] + n0 + 32 * c, whole, left - 32 * c);
                }
            }
        }
    }
    if (ctas > 1) cluster.barrier_wait();        // its own u stays until the others have read it
}

// One row a tile (a decode batch): a fragment of the tensor cores would hold 15 rows of nothing, so the
// products run on the CUDA cores, in fp32 throughout. The cluster's CTAs split K, a warp takes two rank rows
// at a time; then an output is 1, 2 or 4 lanes' work (32 ranks each at most), 4 outputs in flight a lane.
template <bool kFp32>
__global__ void __launch_bounds__(kThreads) adapter_row_kernel(AdapterArgs p) {
    __shared__ __align__(16) float part[kMaxRank], u[kMaxRank];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int unit = blockIdx.x / ctas, t = unit / p.splits, split = unit % p.splits;
    int id = __ldg(p.ids + t);
    if (id < -1 || id >= p.adapters) {
        if (tid == 0 && rank == 0 && split == 0) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
        id = -1;
    }
    const int shares = p.splits * ctas, share = split * ctas + rank, per = ((p.N + shares - 1) / shares + 31) & ~31;
    const int n0 = min(share * per, p.N), n1 = min(n0 + per, p.N);
    const size_t row = (size_t)t * p.N;
    if (id < 0) {                                // the same for the whole cluster; the row keeps its bits
        if (p.out == p.y) return;
        for (int n = n0 + tid; n < n1; n += kThreads) {
            if (kFp32) static_cast<uint32_t *>(p.out)[row + n] = static_cast<const uint32_t *>(p.y)[row + n];
            else static_cast<uint16_t *>(p.out)[row + n] = static_cast<const uint16_t *>(p.y)[row + n];
        }
        return;
    }
    auto dot8 = [](const uint4 &a, const float4 &x, const float4 &z, float s) {
        s = fmaf(__uint_as_float(a.x << 16), x.x, s);
        s = fmaf(__uint_as_float(a.x & 0xffff0000u), x.y, s);
        s = fmaf(__uint_as_float(a.y << 16), x.z, s);
        s = fmaf(__uint_as_float(a.y & 0xffff0000u), x.w, s);
        s = fmaf(__uint_as_float(a.z << 16), z.x, s);
        s = fmaf(__uint_as_float(a.z & 0xffff0000u), z.y, s);
        s = fmaf(__uint_as_float(a.w << 16), z.z, s);
        return fmaf(__uint_as_float(a.w & 0xffff0000u), z.w, s);
    };
    // ---- u = x . A^T
    {
        const int chunks = p.K / 8, each = (chunks + ctas - 1) / ctas;
        const int c0 = rank * each, c1 = min(c0 + each, chunks);
        const uint4 *xr = reinterpret_cast<const uint4 *>(p.x + (size_t)t * p.K);
        for (int j = 2 * warp; j < p.rank; j += 2 * kWarps) {
            const uint4 *a0 = reinterpret_cast<const uint4 *>(p.a + ((size_t)id * p.rank + j) * p.K);
            const uint4 *a1 = a0 + chunks;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
            for (int c = c0 + lane; c < c1; c += 32) {
                const uint4 q = __ldg(xr + c), v0 = __ldg(a0 + c), v1 = __ldg(a1 + c);
                const float4 x = make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u),
                                             __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u));
                const float4 z = make_float4(__uint_as_float(q.z << 16), __uint_as_float(q.z & 0xffff0000u),
                                             __uint_as_float(q.w << 16), __uint_as_float(q.w & 0xffff0000u));
                s0 = dot8(v0, x, z, s0);
                s1 = dot8(v1, x, z, s1);
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) {
                s0 += __shfl_xor_sync(0xffffffffu, s0, off);
                s1 += __shfl_xor_sync(0xffffffffu, s1, off);
            }
            if (lane == 0) {
                part[j] = s0;
                part[j + 1] = s1;
            }
        }
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();
    if (tid < p.rank) {
        float o[kMaxCluster], s = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) o[k] = k < ctas ? *cluster.map_shared_rank(part + tid, k) : 0.f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) s += o[k];
        u[tid] = s * __ldg(p.scale + id);
    }
    __syncthreads();
    if (ctas > 1) cluster.barrier_arrive();      // this CTA has read the others' sums (waited for at the end)
    // ---- out = y + u . B^T
    constexpr int kOut = 4, kQ = 4;              // outputs a lane, chunks of 8 ranks a lane and output
    const int lanes = p.rank <= 32 ? 1 : p.rank <= 64 ? 2 : 4, mine = lane & (lanes - 1), sub = lane / lanes;
    const int step = 32 / lanes, chunks = p.rank / 8;
    for (int b0 = n0 + warp * kOut * step; b0 < n1; b0 += kWarps * kOut * step) {
        uint4 w[kOut][kQ];
        float y[kOut];
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            const int n = b0 + i * step + sub;
            const uint4 *b = reinterpret_cast<const uint4 *>(p.b + ((size_t)id * p.N + n) * p.rank);
#pragma unroll
            for (int c = 0; c < kQ; ++c)
                w[i][c] = n < n1 && mine + c * lanes < chunks ? __ldg(b + mine + c * lanes) : make_uint4(0u, 0u, 0u, 0u);
            y[i] = n >= n1 || mine ? 0.f
                   : kFp32         ? static_cast<const float *>(p.y)[row + n]
                                   : bf16_bits_to_f32(static_cast<const uint16_t *>(p.y)[row + n]);
        }
        float s[kOut] = {};
#pragma unroll
        for (int c = 0; c < kQ; ++c) {
            if (c * lanes >= chunks) break;
            // (a lane behind the last chunk multiplies its zeros by the last one's u, which may not be finite)
            const int at = mine + c * lanes;
            const bool in = at < chunks;
            const float4 x = *reinterpret_cast<const float4 *>(u + 8 * (in ? at : 0));
            const float4 z = *reinterpret_cast<const float4 *>(u + 8 * (in ? at : 0) + 4);
#pragma unroll
            for (int i = 0; i < kOut; ++i) s[i] = in ? dot8(w[i][c], x, z, s[i]) : s[i];
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            for (int off = 1; off < lanes; off <<= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], off);
            const int n = b0 + i * step + sub;
            if (n >= n1 || mine) continue;
            if (kFp32) static_cast<float *>(p.out)[row + n] = y[i] + s[i];
            else static_cast<uint16_t *>(p.out)[row + n] = f32_to_bf16_bits(y[i] + s[i]);
        }
    }
    if (ctas > 1) cluster.barrier_wait();
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + nb && q < p + na;
}

template <typename Kern>
int launch(Kern kern, size_t smem, const AdapterArgs &p, int ctas, cudaStream_t st) {
    if (smem > 48 * 1024)
        MOE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.T + p.rows - 1) / p.rows) * (unsigned)p.splits * (unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 1 : 0;             // (a CTA alone is a cluster of one)
    MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return MOE_OK;
}

template <int kMT, int kNT>
int dispatch_y(const AdapterArgs &p, int ctas, bool fp32, cudaStream_t st) {
    return fp32 ? launch(adapter_kernel<kMT, kNT, true>, sizeof(Smem<kMT, kNT, 3>), p, ctas, st)
                : launch(adapter_kernel<kMT, kNT, false>, sizeof(Smem<kMT, kNT, 2>), p, ctas, st);
}

template <int kMT>
int dispatch_rank(const AdapterArgs &p, int ctas, bool fp32, cudaStream_t st) {
    if (p.rank <= 16) return dispatch_y<kMT, 2>(p, ctas, fp32, st);
    if (p.rank <= 32) return dispatch_y<kMT, 4>(p, ctas, fp32, st);
    if (p.rank <= 64) return dispatch_y<kMT, 8>(p, ctas, fp32, st);
    return dispatch_y<kMT, 16>(p, ctas, fp32, st);
}

}  // namespace

extern "C" int moe_adapter_add(const void *x, int T, int K, int N, const void *a, const void *b, const float *scale,
                               int adapters, int rank, const int32_t *ids, const void *y, int y_fp32, void *out,
                               void *stream) {
    if (!x || !a || !b || !scale || !ids || !y || !out) return moe_set_error(MOE_EINVAL, "adapters: null pointer");
    if (T <= 0 || T > (1 << 24) || K <= 0 || K % 8 || K > (1 << 20) || N <= 0 || N > (1 << 24) || adapters <= 0 ||
        rank <= 0 || rank > kMaxRank || rank % 8)
        return moe_set_error(MOE_EINVAL,
                             "adapters: bad sizes T=%d K=%d N=%d adapters=%d rank=%d (T, N <= 2^24, K <= 2^20; K and "
                             "rank multiples of 8, rank up to %d)", T, K, N, adapters, rank, kMaxRank);
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15)
        return moe_set_error(MOE_EINVAL, "adapters: x, a and b must be 16-byte aligned");
    const size_t es = y_fp32 ? 4 : 2, ny = (size_t)T * N * es;
    const uintptr_t ya = reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out);
    if (ya & (es - 1)) return moe_set_error(MOE_EINVAL, "adapters: y and out must be aligned to their %zu-byte values", es);
    if ((out != y && overlap(out, ny, y, ny)) || overlap(out, ny, x, (size_t)T * K * 2) ||
        overlap(out, ny, a, (size_t)adapters * rank * K * 2) || overlap(out, ny, b, (size_t)adapters * rank * N * 2) ||
        overlap(out, ny, scale, (size_t)adapters * 4) || overlap(out, ny, ids, (size_t)T * 4))
        return moe_set_error(MOE_EINVAL, "adapters: out may be y itself, but not overlap it or another input");
    AdapterArgs p{static_cast<const uint16_t *>(x), T, K, N, static_cast<const uint16_t *>(a),
                  static_cast<const uint16_t *>(b), scale, adapters, rank, ids, y, out, 16, 1, 0,
                  (ya & 15) == 0 && ((size_t)N * es) % 16 == 0};
    const int full = 296;              // two CTAs on each of 148 SMs
    // One row a tile while reading each row's own A and B costs less than what tiles cost on top: a decode
    // batch, or up to 32 MB of them (K = 3,072, N = 768, rank 16, 30 adapters: 5.3 us against 8.6 for 100
    // rows, 7.2 against 11.7 for 300; rank 64 of 2,048 x 2,048: 20 against 11.4 for 150). A batch of up to 74
    // rows goes by rows whatever its width, where several adapters would each be a tile's: fp32 y of 248,320,
    // 64 rows, rank 16 120 us against 167 with 8 adapters (99 with one for all), rank 64 333 against 429 (232),
    // rank 128 638 against 1,157 (589). A cluster a row only where there are few (one row: 4.0 us with
    // 8 CTAs, 64 rows: 5.0 with 1, 5.3 with 4).
    const bool single = T <= full / 4 || (double)T * rank * ((double)K + N) * 2 <= 32e6;
    int ctas;
    if (single) {
        p.rows = 1;
        ctas = T * 8 <= full ? kMaxCluster : T < 64 ? 4 : 1;
    } else {
        // as few rows a tile as leave two CTAs an SM at four CTAs a tile, since the phases of a tile follow
        // one another and only more tiles hide that (2,048 rows of rank 64: 26 us with 32 rows, 31 with 16)
        p.rows = 2;
        while (p.rows < 32 && (long long)((T + p.rows - 1) / p.rows) * 4 > full) p.rows *= 2;
        ctas = (T + p.rows - 1) / p.rows * 8 <= full ? kMaxCluster : (T + p.rows - 1) / p.rows * 4 <= 2 * full ? 4 : 2;
    }
    // a wide N (an LM head) is split over clusters of two, which repeat the small first product
    const int tiles = (T + p.rows - 1) / p.rows;
    if (N >= 16384 && ctas > 2) ctas = 2;
    while ((long long)tiles * ctas * (p.splits + 1) <= full && N / (ctas * (p.splits + 1)) >= kWarps * 64) ++p.splits;
    const bool wide = p.rows > 16;
    if (single)
        return y_fp32 ? launch(adapter_row_kernel<true>, 0, p, ctas, as_stream(stream))
                      : launch(adapter_row_kernel<false>, 0, p, ctas, as_stream(stream));
    p.sort = p.rows > 1 && T > p.rows && adapters <= kMaxSort;
    return wide ? dispatch_rank<2>(p, ctas, y_fp32 != 0, as_stream(stream))
                : dispatch_rank<1>(p, ctas, y_fp32 != 0, as_stream(stream));
}
