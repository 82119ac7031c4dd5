// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = y[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T,   a = ids[t]   (a = -1: out[t] = y[t])
//
// with A [adapters, rank, K], B [adapters, N, rank] bf16 and y the projection's own output (bf16,
// or the LM head's fp32 logits). One launch, no workspace: a cluster of CTAs takes a tile of rows and
// a range of the N outputs. First u = x . A^T: the cluster's CTAs split K, their warps split it again,
// and the partial sums (fp32) are added in a fixed order through distributed shared memory. Then each
// CTA adds u . B^T to its share of the outputs. A tile goes through the adapters that its rows name, one
// after another; rows of other adapters ride along in the products and are left out of the results,
// so ids may come in any order.
//
// The products are 8 to 128 wide, far too little arithmetic per byte to be bound by the tensor cores
// (rank 64: 60 FLOP per byte of x, y and out): mma.sync takes its operands from registers,
// straight from 16-byte global loads. For that the K order inside a step is permuted alike in both
// operands: a lane's consecutive elements fill its places of the fragments.
//
// u is carried into the second product as two bf16 (u = hi + lo, off by 2^-17 of u at most): the fp32
// logits of an adapted head must not lose digits that one bf16 would drop.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxRank = 128, kMaxCluster = 8;
constexpr int kGroup = 32;             // outputs a warp takes at a time: 4 fragments of 8

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
};

MOE_D void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

MOE_D uint32_t pack_bf16(float a, float b) {
    return (uint32_t)f32_to_bf16_bits(a) | ((uint32_t)f32_to_bf16_bits(b) << 16);
}

// what a bf16 drops of v; nothing of what is not finite
MOE_D float below_bf16(float v) {
    const float r = bf16r(v);
    return fabsf(r) < INFINITY ? v - r : 0.f;
}

// kMT: row fragments (16 rows) a tile; kNT: fragments of 8 rank rows the warps have registers for
template <int kMT, int kNT>
struct Smem {
    static constexpr int kRows = 16 * kMT, kWK = kWarps / kMT;       // warps along K per row fragment
    static constexpr int kR = 8 * kNT, kSteps = (kR + 15) / 16;
    float part[kWK][kRows][kR];        // the warps' sums over their K steps
    float u[kRows][kR];                // the CTA's sums, read by the cluster
    uint4 frag[2][kMT][kSteps][32];    // scale * u as fragments: high and low parts
    int id[kRows], kind[kRows];        // the rows' adapters; the different ones among them
    unsigned long long member[kRows];  // which rows are of that kind
    int kinds;
};

template <bool kFp32, bool kVec>
MOE_D void load8(const void *y, size_t at, int left, float (&v)[8]) {
    if (kVec && left >= 8) {
        if (kFp32) {
            const float4 p = *reinterpret_cast<const float4 *>(static_cast<const float *>(y) + at);
            const float4 q = *reinterpret_cast<const float4 *>(static_cast<const float *>(y) + at + 4);
            v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
        } else {
            const uint4 p = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(y) + at);
            const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i >= left ? 0.f : kFp32 ? static_cast<const float *>(y)[at + i]
                                           : bf16_bits_to_f32(static_cast<const uint16_t *>(y)[at + i]);
    }
}

template <bool kFp32, bool kVec>
MOE_D void store8(void *out, size_t at, int left, const float (&v)[8]) {
    if (kVec && left >= 8) {
        if (kFp32) {
            float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
            o[0] = make_float4(v[0], v[1], v[2], v[3]);
            o[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) = make_uint4(
                pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= left) break;
            if (kFp32) static_cast<float *>(out)[at + i] = v[i];
            else static_cast<uint16_t *>(out)[at + i] = f32_to_bf16_bits(v[i]);
        }
    }
}

// kVec: rows of y and out start at 16-byte boundaries
template <int kMT, int kNT, bool kFp32, bool kVec>
__global__ void __launch_bounds__(kThreads) adapter_kernel(AdapterArgs p) {
    using S = Smem<kMT, kNT>;
    extern __shared__ __align__(16) unsigned char smem[];
    S &sh = *reinterpret_cast<S *>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int unit = blockIdx.x / ctas, tile = unit / p.splits, split = unit % p.splits;
    const int t0 = tile * p.rows, rows = min(p.rows, p.T - t0);

    // ---- the adapters of the tile, in the order of their first rows
    if (tid < S::kRows) {
        int id = tid < rows ? p.ids[t0 + tid] : -1;
        if (id < -1 || id >= p.adapters) {
            if (rank == 0 && split == 0) atomicOr(&g_moe_device_error, MOE_DEVERR_BAD_INPUT);
            id = -1;
        }
        sh.id[tid] = id;
    }
    __syncthreads();
    if (warp == 0) {
        int n = 0;
#pragma unroll
        for (int h = 0; h < S::kRows; h += 32) {
            const int r = h + lane;
            const int id = r < S::kRows ? sh.id[r] : -1;
            unsigned long long same = 0ull;
#pragma unroll 1
            for (int j = 0; j < S::kRows; ++j) same |= (unsigned long long)(sh.id[j] == id) << j;
            const bool first = id >= 0 && __ffsll((long long)same) - 1 == r;
            const unsigned who = __ballot_sync(0xffffffffu, first);
            if (first) {
                const int at = n + __popc(who & ((1u << lane) - 1u));
                sh.kind[at] = id;
                sh.member[at] = same;
            }
            n += __popc(who);
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
        const uint16_t *xa = p.x + (size_t)(t0 + ra) * p.K + 8 * q, *xb = p.x + (size_t)(t0 + rb) * p.K + 8 * q;
        const bool oka = ra < rows, okb = rb < rows;
        for (int d = 0; d < kinds; ++d) {
            if (!((sh.member[d] >> (16 * mt)) & 0xffffull)) continue;             // none of this warp's rows
            const uint16_t *ar = p.a + ((size_t)sh.kind[d] * p.rank + g) * p.K + 8 * q;
            float acc[kNT][4] = {};
#pragma unroll 2
            for (int s = rank * per + wk; s < s1; s += S::kWK) {
                const bool in = 32 * s + 8 * q < p.K;
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                const uint4 va = in && oka ? *reinterpret_cast<const uint4 *>(xa + 32 * s) : zero;
                const uint4 vb = in && okb ? *reinterpret_cast<const uint4 *>(xb + 32 * s) : zero;
                uint4 w[kNT];
#pragma unroll
                for (int j = 0; j < kNT; ++j)
                    w[j] = in && j < nt ? __ldg(reinterpret_cast<const uint4 *>(ar + (size_t)8 * j * p.K + 32 * s)) : zero;
#pragma unroll
                for (int j = 0; j < kNT; ++j) {
                    mma16816(acc[j], va.x, vb.x, va.y, vb.y, w[j].x, w[j].y);
                    mma16816(acc[j], va.z, vb.z, va.w, vb.w, w[j].z, w[j].w);
                }
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
        if (sh.id[r] >= 0) {
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
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * m + (l >> 2) + 8 * h;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < S::kR && sh.id[r] >= 0) {
                for (int k = 0; k < ctas; ++k) {
                    const float4 o = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(&sh.u[r][c], k));
                    v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                }
                const float f = __ldg(p.scale + sh.id[r]);
                v.x *= f; v.y *= f; v.z *= f; v.w *= f;
            }
            hi[h] = pack_bf16(v.x, v.y);
            hi[2 + h] = pack_bf16(v.z, v.w);
            lo[h] = pack_bf16(below_bf16(v.x), below_bf16(v.y));
            lo[2 + h] = pack_bf16(below_bf16(v.z), below_bf16(v.w));
        }
        sh.frag[0][m][s][l] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        sh.frag[1][m][s][l] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (ctas > 1) cluster.sync();                // (the others have read this CTA's u)
    else __syncthreads();

    // ---- out = y + u . B^T, 32 outputs a warp at a time: fragment f, place (q, e) is output
    // n0 + 8 q + 2 f + e, so that a lane ends with 8 consecutive ones
    const int groups = (p.N + kGroup - 1) / kGroup, shares = p.splits * ctas;
    const int share = split * ctas + rank;
    const int gper = (groups + shares - 1) / shares, g1 = min((share + 1) * gper, groups);
    const int steps = (p.rank + 15) / 16;
    for (int gr = share * gper + warp; gr < g1; gr += kWarps) {
        const int n0 = gr * kGroup, left = p.N - (n0 + 8 * q);
        float acc[kMT][4][4] = {};
        for (int d = 0; d < kinds; ++d) {
            const unsigned long long member = sh.member[d];
            // fragment column g of fragment f: output n0 + 8 (g / 2) + 2 f + g % 2
            const int nb = n0 + 8 * (g >> 1) + (g & 1);
            const uint16_t *br = p.b + ((size_t)sh.kind[d] * p.N + nb) * p.rank + 4 * q;
            float sum[kMT][4][4] = {};
#pragma unroll 2
            for (int s = 0; s < steps; ++s) {
                uint2 w[4];
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    w[f] = nb + 2 * f < p.N && 16 * s + 4 * q < p.rank
                               ? __ldg(reinterpret_cast<const uint2 *>(br + (size_t)2 * f * p.rank + 16 * s))
                               : make_uint2(0u, 0u);
#pragma unroll
                for (int m = 0; m < kMT; ++m) {
                    if (kMT > 1 && !((member >> (16 * m)) & 0xffffull)) continue;
                    const uint4 hi = sh.frag[0][m][s][lane], lo = sh.frag[1][m][s][lane];
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        mma16816(sum[m][f], hi.x, hi.y, hi.z, hi.w, w[f].x, w[f].y);
                        mma16816(sum[m][f], lo.x, lo.y, lo.z, lo.w, w[f].x, w[f].y);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < kMT; ++m) {
                const bool ma = (member >> (16 * m + g)) & 1ull, mb = (member >> (16 * m + g + 8)) & 1ull;
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    if (ma) { acc[m][f][0] = sum[m][f][0]; acc[m][f][1] = sum[m][f][1]; }
                    if (mb) { acc[m][f][2] = sum[m][f][2]; acc[m][f][3] = sum[m][f][3]; }
                }
            }
        }
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 16 * m + g + 8 * h;
                if (r >= rows || left <= 0) continue;
                const size_t at = (size_t)(t0 + r) * p.N + n0 + 8 * q;
                float v[8];
                load8<kFp32, kVec>(p.y, at, left, v);
                if (sh.id[r] >= 0) {                                // (a kept row keeps its bits, NaN too)
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        v[2 * f] += acc[m][f][2 * h];
                        v[2 * f + 1] += acc[m][f][2 * h + 1];
                    }
                }
                store8<kFp32, kVec>(p.out, at, left, v);
            }
    }
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + nb && q < p + na;
}

template <int kMT, int kNT, bool kFp32, bool kVec>
int launch(const AdapterArgs &p, int ctas, cudaStream_t st) {
    auto kern = adapter_kernel<kMT, kNT, kFp32, kVec>;
    const size_t smem = sizeof(Smem<kMT, kNT>);
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
    cfg.numAttrs = 1;
    MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return MOE_OK;
}

template <int kMT, int kNT>
int dispatch_y(const AdapterArgs &p, int ctas, bool fp32, bool vec, cudaStream_t st) {
    if (fp32) return vec ? launch<kMT, kNT, true, true>(p, ctas, st) : launch<kMT, kNT, true, false>(p, ctas, st);
    return vec ? launch<kMT, kNT, false, true>(p, ctas, st) : launch<kMT, kNT, false, false>(p, ctas, st);
}

template <int kMT>
int dispatch_rank(const AdapterArgs &p, int ctas, bool fp32, bool vec, cudaStream_t st) {
    if (p.rank <= 16) return dispatch_y<kMT, 2>(p, ctas, fp32, vec, st);
    if (p.rank <= 32) return dispatch_y<kMT, 4>(p, ctas, fp32, vec, st);
    if (p.rank <= 64) return dispatch_y<kMT, 8>(p, ctas, fp32, vec, st);
    return dispatch_y<kMT, 16>(p, ctas, fp32, vec, st);
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
                  static_cast<const uint16_t *>(b), scale, adapters, rank, ids, y, out, 16, 1};
    int ctas = kMaxCluster;
    const bool vec = (ya & 15) == 0 && ((size_t)N * es) % 16 == 0;
    const bool wide = T >= 512;
    if (wide) {
        p.rows = 64;
        ctas = 4;
    } else {
        // enough clusters for all SMs: split N while a warp keeps a group, then take fewer rows a tile
        const int tiles = (T + 15) / 16, want = 37;
        while (p.splits * tiles < want && N / (p.splits + 1) >= ctas * kWarps * kGroup) ++p.splits;
        const int rows = (int)(((long long)T * p.splits * ctas + 147) / 148);
        p.rows = rows < 16 ? rows : 16;
    }
    return wide ? dispatch_rank<4>(p, ctas, y_fp32 != 0, vec, as_stream(stream))
                : dispatch_rank<1>(p, ctas, y_fp32 != 0, vec, as_stream(stream));
}
