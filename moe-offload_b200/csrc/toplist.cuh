// Row statistics of a softmax and the n largest entries of a row, as the log-probability
// kernels (logprobs.cu, headscore.cu) keep them.
#pragma once

#include "common.cuh"

constexpr int kTopMax = 32;            // alternatives a row can be asked for: one per lane of a warp

// Softmax statistics over a set of values x: m the largest, s = sum e^(x - m) over the set
// WITHOUT one occurrence of m, w = sum (x - m) e^(x - m). Keeping the largest out of s keeps the
// digits of rows whose probability is all but one: lse - m = log1p(s), and s itself is then far
// below the rounding of 1 + s. Nothing yet: m = -inf. A NaN among the values ends up in s; a row
// whose m is not finite has no distribution (soft_log_rest is NaN).
struct Soft {
    float m, s, w;
};

// e^kSoftFar is 0 in fp32: differences are held above it, so that 0 x inf does not arise for masked
// (-inf) or lowest-value logits
constexpr float kSoftFar = -1000.f;

// e^x and 2^x by the exponential unit, results below the smallest normal number 0 (without that, every
// call carries three more instructions for them). The product with log2(e) is rounded: e^x is off by
// |x| 2^-24 and more, alike for no two values, which a sum of many evens out. What scales a whole sum
// takes expf.
MOE_D float fast_pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;
MOE_D float fast_exp(float x) { return fast_pow2(x * kLog2e); }

MOE_D Soft soft_none() { return Soft{-INFINITY, 0.f, 0.f}; }

MOE_D Soft soft_merge(Soft a, Soft b) {
    if (a.m < b.m) { const Soft t = a; a = b; b = t; }
    if (b.m == -INFINITY) {                      // nothing there (s is 0, or NaN to be passed on)
        a.s += b.s;
        return a;
    }
    const float d = fmaxf(b.m - a.m, kSoftFar), e = expf(d);
    a.w += e * (b.w + d * (b.s + 1.f));
    a.s += (b.s + 1.f) * e;
    return a;
}

// lse - m, NaN for a row without a distribution
MOE_D float soft_log_rest(const Soft &a) {
    return (a.m < INFINITY && a.m > -INFINITY) ? log1pf(a.s) : __int_as_float(0x7fffffff);
}

// entropy in nats: lse - sum p x = log1p(s) - w / (1 + s)
MOE_D float soft_entropy(const Soft &a) { return soft_log_rest(a) - a.w / (1.f + a.s); }

MOE_D Soft soft_shfl_xor(const Soft &a, int off) {
    return Soft{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                __shfl_xor_sync(0xffffffffu, a.w, off)};
}

MOE_D Soft soft_warp(Soft a) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Soft b = soft_shfl_xor(a, off);
        // both lanes of a pair merge in the same order, so that every lane ends with the same bits
        a = (threadIdx.x & off) ? soft_merge(b, a) : soft_merge(a, b);
    }
    return a;
}

// The same statistics while a thread runs over its values: sums relative to a reference r that
// stays within kRunSpan below the largest value m, so that most steps neither rescale nor branch.
// The sums hold every value but the largest: a new value v adds min(m, v) and leaves max(m, v) out.
struct SoftRun {
    float m, r, s, w;
};
constexpr float kRunSpan = 32.f;       // e^32 * 2^30 values stay far inside fp32

// the smaller of two, NaN if either is one
MOE_D float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

MOE_D SoftRun run_none() { return SoftRun{-INFINITY, 0.f, 0.f, 0.f}; }

// Adds kN values; top: the largest of them and of all before (NaN left out).
template <int kN>
MOE_D void run_add(SoftRun &a, const float (&v)[kN], float top) {
    if (top > a.m && !(top <= a.r + kRunSpan && a.m > -INFINITY)) {
        const float d = fmaxf(a.r - top, kSoftFar), f = a.m > -INFINITY ? expf(d) : 1.f;
        a.w = f * (a.w + d * a.s);
        a.s *= f;                                // (nothing in the sums yet: 0, or NaN)
        a.r = top;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const float d = min_nan(a.m, v[i]) - a.r, e = fast_exp(d);     // e^-inf = 0, NaN stays
        a.m = fmaxf(a.m, v[i]);
        a.s += e;
        a.w = fmaf(fmaxf(d, kSoftFar), e, a.w);
    }
}

// ------------------------------------------------------------------ order of the entries

// Order-preserving 64-bit key of (value, index): larger value first, equal values the lower
// index first. 0 is no entry. NaN orders as -inf, -0 as +0.
MOE_D unsigned long long top_key(float v, int idx) {
    v = v != v ? -INFINITY : v + 0.f;
    const uint32_t u = __float_as_uint(v);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)o << 32) | (unsigned long long)(0xffffffffu - (uint32_t)idx);
}
MOE_D float top_value(unsigned long long k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
MOE_D int top_index(unsigned long long k) { return (int)(0xffffffffu - (uint32_t)(k & 0xffffffffull)); }

// A step of a bitonic network over one key per lane.
MOE_D unsigned long long top_cmpx(unsigned long long k, int off, bool keep_max) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, off);
    return (k > o) == keep_max ? k : o;
}
// a, b sorted descending over the lanes: the 32 largest of both, sorted descending
MOE_D unsigned long long top_merge(unsigned long long a, unsigned long long b) {
    const int lane = threadIdx.x & 31;
    b = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a > b ? a : b;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) a = top_cmpx(a, off, (lane & off) == 0);
    return a;
}
// inserts a key that all lanes hold into a sorted list
MOE_D unsigned long long top_insert(unsigned long long list, unsigned long long key) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
    // entries above the key stay, the others move down by one, the key takes the gap
    return list > key ? list : ((threadIdx.x & 31) == 0 || up > key) ? key : up;
}
