// Log probabilities of given tokens, the entropy of each row and its most likely alternatives, from logits [rows][vocab];
// and the gradient of the first two.
//
//   m = max_j x_j,  s = sum_j e^(x_j - m),  log p_j = (x_j - m) - log s
//   H = -sum_j p_j log p_j = log s - (1/s) sum_j (x_j - m) e^(x_j - m)
//   dx_j = dlp (1[j = token] - p_j) - dH p_j (log p_j + H)
//
// One pass over the logits: every thread keeps a running maximum with the two sums against it and rescales them when
// the maximum grows.  The reference has no counterpart beyond its softmax and cross-entropy kernels
// (nectarml/csrc/kernels/tensor/fused/), which write the whole distribution.
//
// What bounds it.  Memory: 2 or 4 bytes a logit.  An fp16 logit at the memory's rate leaves an SM 10.7 instructions of a lane and 1.3 of its
// special function unit, so the inner loop is short: powers of two (the logits times log2 e, less that of the maximum, in one FMA) and pairs of
// fp32 operations in one instruction; 4.5 instructions and one power a logit.
//
// Units.  A row is read in units of 32 bytes (one load of 256 bits) that start on 32-byte boundaries of memory, so a row of an
// odd vocabulary, which starts anywhere, is read like any other; its first and last unit are taken element by element.
//
// Alternatives.  The pass also notes the largest logit of every unit.  Let t be the `top`-th largest among the maxima of 128 groups of
// units: at least `top` logits are t or more, so only units whose maximum is that are read again, and of their logits only those; each of them
// then counts those that come before it, which is its place.  The row is not searched.  Where ties make that too many (a row that is
// masked as a whole), the largest unit is taken `top` times instead.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/nectarml_b200.h"
#include "nml_host.cuh"
#include "nml_launch.cuh"

namespace nml_logits {

using nml::load_global;
using nml::pdl_enter;

#define NMLG_CUDA(expr)                                                             \
    do {                                                                            \
        const cudaError_t e_ = (expr);                                              \
        if (e_ != cudaSuccess) return nml::cuda_failed(static_cast<int>(e_), #expr); \
    } while (0)

constexpr int kMaxTop = 32;          // a lane to each
constexpr int kUnitBytes = 32;
constexpr int kGroups = 128;         // of units, for the search
constexpr int kMaxUnits = 127 * kGroups;  // of one block's share of a row: its maxima take 63.5 KB
constexpr int kMaxCluster = 8;
constexpr int kWarpRows = 4;         // rows of a warp each, to a block
constexpr int kChosen = 256, kCandidates = 512;  // units and logits of the search

__device__ __forceinline__ void load_unit(const void* p, uint32_t (&v)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(__cvta_generic_to_global(p)));
}
__device__ __forceinline__ void store_unit(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ long long load_index(const long long* p) {
    long long v;
    asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(__cvta_generic_to_global(p)));
    return v;
}

// Two fp32 values in one register pair.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ float low(uint64_t v) { return unpack2(v).x; }
__device__ __forceinline__ float high(uint64_t v) { return unpack2(v).y; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^y, 0 below 2^-126; two units in the last place.
__device__ __forceinline__ float power2(float y) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    return e;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

template <typename T>
struct Elements;
template <>
struct Elements<float> {
    static constexpr int N = 8;
    // Largest of a unit; NaN where it has one.
    static __device__ __forceinline__ float largest(const uint32_t (&v)[8]) {
        float m = __uint_as_float(v[0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) m = max_nan(m, __uint_as_float(v[j]));
        return m;
    }
    // As pairs, with what is masked (-inf, or the lowest value) at a finite distance.
    static __device__ __forceinline__ void pairs(const uint32_t (&v)[8], uint64_t (&x)[N / 2]) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) x[j] = pack2(fmaxf(__uint_as_float(v[2 * j]), -1e32f), fmaxf(__uint_as_float(v[2 * j + 1]), -1e32f));
    }
    static __device__ __forceinline__ float get(const uint32_t (&v)[8], int j) { return __uint_as_float(v[j]); }
    static __device__ __forceinline__ float of(uint2 v, int j) { return __uint_as_float(j ? v.y : v.x); }
    static __device__ __forceinline__ void pack(const uint64_t (&x)[N / 2], uint32_t (&v)[8]) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) v[2 * j] = __float_as_uint(low(x[j])), v[2 * j + 1] = __float_as_uint(high(x[j]));
    }
    static __device__ __forceinline__ float load(const float* p) { return load_global(p); }
    static __device__ __forceinline__ float round(float x) { return x; }
};
template <>
struct Elements<__half> {
    static constexpr int N = 16;
    static __device__ __forceinline__ __half2 at(const uint32_t (&v)[8], int j) { return *reinterpret_cast<const __half2*>(&v[j]); }
    static __device__ __forceinline__ float largest(const uint32_t (&v)[8]) {
        __half2 m = at(v, 0);
#pragma unroll
        for (int j = 1; j < 8; ++j) m = __hmax2_nan(m, at(v, j));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void pairs(const uint32_t (&v)[8], uint64_t (&x)[N / 2]) {
        const __half2 lowest = __half2half2(__ushort_as_half(0xfbff));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = __half22float2(__hmax2(at(v, j), lowest));
            x[j] = pack2(f.x, f.y);
        }
    }
    static __device__ __forceinline__ float get(const uint32_t (&v)[8], int j) {
        return j & 1 ? __high2float(at(v, j / 2)) : __low2float(at(v, j / 2));
    }
    static __device__ __forceinline__ float of(uint2 v, int j) {
        const uint32_t w = j & 2 ? v.y : v.x;
        const __half2 h = *reinterpret_cast<const __half2*>(&w);
        return j & 1 ? __high2float(h) : __low2float(h);
    }
    static __device__ __forceinline__ void pack(const uint64_t (&x)[N / 2], uint32_t (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2 h = __floats2half2_rn(low(x[j]), high(x[j]));
            v[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(load_global(p)); }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};

// Floats in the order of unsigned integers (-0 and 0 are one value; NaN above everything).  0 is below every float: "none".
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A row as units: unit u holds the elements u * N - lead ... of which those in [0, vocab) exist.
template <typename T>
struct Row {
    static constexpr int N = Elements<T>::N;
    const T* base;  // of unit 0: at or before the row's first element, on a 32-byte boundary
    int lead, vocab, units;
    int full0, full1;  // units without a gap
    __device__ __forceinline__ Row(const T* row, int vocab_) {
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) & (kUnitBytes - 1)) / sizeof(T));
        base = row - lead;
        vocab = vocab_;
        const long long end = static_cast<long long>(lead) + vocab;
        units = static_cast<int>((end + N - 1) / N);
        full0 = lead ? 1 : 0;
        full1 = static_cast<int>(end / N);
    }
    __device__ __forceinline__ const T* at(int u) const { return base + static_cast<long long>(u) * N; }
    __device__ __forceinline__ long long first(int u) const { return static_cast<long long>(u) * N - lead; }
    __device__ __forceinline__ bool has(long long i) const { return i >= 0 && i < vocab; }
    // The bits of a unit with gaps; those of -inf in them.
    __device__ __forceinline__ void load_broken(int u, uint32_t (&v)[8]) const {
        uint32_t w[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float x = has(first(u) + j) ? Elements<T>::load(at(u) + j) : -INFINITY;
            w[j] = sizeof(T) == 4 ? __float_as_uint(x) : static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x)));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = sizeof(T) == 4 ? w[j % N] : w[2 * j % N] | w[(2 * j + 1) % N] << 16;
    }
};

// Running statistics: the maximum m, and against 2^M, M = m log2 e rounded, the sums of 2^y and y 2^y with y = x log2 e - M.
// While everything is -inf, m is -inf and the sums are 0.  Where m is no number or infinite, so is the row, and the sums do not matter.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Where a maximum leaves no room below it for what is masked (fp16: near the lowest value), or is so large that the product with log2 e is rounded by
// more than a half (and 2 to the power of that is soon no finite number), logits are taken by their distance from m, which is then the reference itself.
template <typename T>
__device__ __forceinline__ bool extreme(float m) { return sizeof(T) == 4 ? !(fabsf(m) < 1e7f) : m < -65000.f; }
template <typename T>
__device__ __forceinline__ float reference(float m) { return extreme<T>(m) ? 0.f : __fmul_rn(m, kLog2e); }  // (rounded wherever it stands)
constexpr float kFar = -1e20f;  // instead of a distance of -inf; times the largest sums, 2^31 logits of e^kSlack, a finite number

struct Stats {
    float m, s, t;
};
// What the reference of m lies below m log2 e.
template <typename T>
__device__ __forceinline__ float below(float m) { return extreme<T>(m) ? 0.f : fmaf(m, kLog2e, -reference<T>(m)); }
// How far y moves where the maximum a becomes b >= a: from one reference to the other.  Where only one of them is rounded, by what that one
// lacks too, which is up to a half: 2^0.5 in the sums of a row whose maxima lie on both sides of 1e7.
template <typename T>
__device__ __forceinline__ float moved_by(float a, float b) {
    const bool far_a = extreme<T>(a), far_b = extreme<T>(b);
    if (!far_a && !far_b) return reference<T>(a) - reference<T>(b);
    return fmaxf(fmaf(a - b, kLog2e, below<T>(b) - below<T>(a)), kFar);
}
// The statistics of the lanes of a warp (or of its first `width`), in every lane: against the largest maximum, once, then two plain sums.  `m` is the
// lane's maximum where a.m is another reference.
template <typename T>
__device__ __forceinline__ Stats merge_lanes(Stats a, int width, float m) {
    for (int o = width / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float d = a.s != 0.f ? moved_by<T>(a.m, m) : 0.f, f = power2(d);
    a.t = (a.t + d * a.s) * f;
    a.s *= f;
    for (int o = width / 2; o > 0; o /= 2) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    a.m = m;
    return a;
}
template <typename T>
__device__ __forceinline__ Stats merge_lanes(const Stats& a, int width) { return merge_lanes<T>(a, width, a.m); }

// A thread's own, the sums over even and odd elements apart.  They stand against `from`, a maximum that was, and move only where the new one is
// more than kSlack above it: a lane in 32 has a new maximum nearly always (30 of 32 units of a row of random logits; the moves were 3.5 of 8.1
// instructions a logit), and sums of up to 2^24 times e^kSlack are as exact as of 1.
constexpr float kSlack = 8.f;
template <typename T>
struct Running {
    float m = -INFINITY, from = -INFINITY, limit = -INFINITY, M = 0.f;
    uint64_t s = 0, t = 0;

    // -> the unit's largest
    __device__ __forceinline__ float add(const uint32_t (&v)[8]) {
        constexpr int N = Elements<T>::N;
        const float most = Elements<T>::largest(v);
        m = max_nan(m, most);
        if (!(most <= limit)) {
            const float d = s != 0 ? moved_by<T>(from, m) : 0.f, f = power2(d);
            t = mul2(fma2(pack2(d, d), s, t), pack2(f, f));
            s = mul2(s, pack2(f, f));
            from = m;
            limit = m + kSlack;
            M = reference<T>(m);
        }
        if (extreme<T>(from) && from != -INFINITY) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float y = fmaxf((Elements<T>::get(v, j) - from) * kLog2e, kFar), e = power2(y);
                s = add2(s, pack2(e, 0.f));
                t = add2(t, pack2(y * e, 0.f));
            }
            return most;
        }
        uint64_t x[N / 2];
        Elements<T>::pairs(v, x);
        const uint64_t k = pack2(kLog2e, kLog2e), r = pack2(-M, -M);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const uint64_t y = fma2(x[j], k, r), e = pack2(power2(low(y)), power2(high(y)));
            s = add2(s, e);
            t = fma2(y, e, t);
        }
        return most;
    }
    __device__ __forceinline__ Stats done() const { return merge_lanes<T>({from, low(s) + high(s), low(t) + high(t)}, 32, m); }  // of the warp
};

// One block's part of the search, and a cluster's exchange.
struct Shared {
    Stats warp[8], block;
    alignas(16) uint32_t group[kGroups];  // (read as vectors)
    uint32_t threshold;
    int units, candidates;
    int unit[kChosen];
    alignas(16) uint64_t candidate[kCandidates];
    uint64_t best[kMaxTop];  // the block's alternatives, in order; 0: fewer
};

template <int kThreads>
__device__ __forceinline__ void block_sync() {
    if (kThreads == 32) __syncwarp(); else __syncthreads();
}

// An element as a number: by value, then the lower index first; 0: none.
__device__ __forceinline__ uint64_t candidate(uint32_t key, long long index) { return key ? static_cast<uint64_t>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(index)) : 0; }
__device__ __forceinline__ float value_of(uint64_t c) { return key_value(static_cast<uint32_t>(c >> 32)); }
__device__ __forceinline__ int index_of(uint64_t c) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(c)); }

// Places of `count` candidates (all different): the first `top` go to best.
template <int kThreads>
__device__ __forceinline__ void place(uint64_t* candidates, int count, int top, uint64_t* best) {
    for (int c = threadIdx.x; c < count; c += kThreads) {
        const uint64_t mine = candidates[c];
        int before = 0;
#pragma unroll 4
        for (int o = 0; o < count / 2; ++o) {
            const ulonglong2 v = reinterpret_cast<const ulonglong2*>(candidates)[o];
            before += (v.x > mine) + (v.y > mine);
        }
        if (count & 1) before += candidates[count - 1] > mine;
        if (before < top && mine != 0) best[before] = mine;
    }
}

// The largest unit, `top` times: for rows with so many ties that the search below finds no short list.  One warp; takes the maxima of the
// units that it chooses away.
template <typename T>
__device__ __forceinline__ void search_units(const Row<T>& row, int first, int n, int per, int top, uint32_t* maxima, Shared& sh) {
    const int lane = threadIdx.x & 31;
    constexpr int kMine = kGroups / 32, N = Elements<T>::N;
    uint32_t group[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) group[j] = sh.group[lane * kMine + j];
    int found = 0;
    uint32_t last = 0;
    for (; found < top; ++found) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int j = kMine - 1; j >= 0; --j)
            if (group[j] >= best) best = group[j], at = j;
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;  // fewer units than alternatives
        last = most;
        const int owner = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
        const int lo = __shfl_sync(0xffffffffu, lane * kMine + at, owner) * per, hi = min(n, lo + per);
        // its first unit with that maximum, and its maximum without that unit
        uint32_t unit = 0xffffffffu, rest = 0;
        for (int u = lo + lane; u < hi; u += 32)
            if (maxima[u] == most) unit = min(unit, static_cast<uint32_t>(u));
        unit = __reduce_min_sync(0xffffffffu, unit);
        for (int u = lo + lane; u < hi; u += 32)
            if (u != static_cast<int>(unit)) rest = max(rest, maxima[u]);
        rest = __reduce_max_sync(0xffffffffu, rest);
        __syncwarp();
        if (lane == 0) {
            maxima[unit] = 0;
            sh.unit[found] = static_cast<int>(unit);
        }
        if (lane == owner) {
#pragma unroll
            for (int j = 0; j < kMine; ++j)
                if (j == at) group[j] = rest;
        }
        __syncwarp();
    }
    if (found < top) last = 1;
    // their elements that are as large as the last one's, at most 32 x 16
    int count = 0;
#pragma unroll 4
    for (int e0 = 0; e0 < found * N; e0 += 32) {
        const int e = e0 + lane, u = first + (e < found * N ? sh.unit[e / N] : 0);
        const long long i = row.first(u) + e % N;
        const uint32_t k = e < found * N && row.has(i) ? order_key(Elements<T>::load(row.at(u) + e % N)) : 0;
        const bool in = k != 0 && k >= last;
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (in) {
            sh.candidate[count + __popc(who & ((1u << lane) - 1))] = candidate(k, i);
        }
        count += __popc(who);
    }
    __syncwarp();
    place<32>(sh.candidate, count, top, sh.best);
    __syncwarp();
}

// The top-th largest of the groups' maxima, as the threshold: one warp takes the largest away, as often.
__device__ __forceinline__ void largest_groups(int top, Shared& sh) {
    const int tid = threadIdx.x;
    if (tid >= 32) return;
    constexpr int kMine = kGroups / 32;
    uint32_t group[kMine], most = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) group[j] = sh.group[j * 32 + tid];
    for (int k = 0; k < top; ++k) {
        uint32_t mine = group[0];
#pragma unroll
        for (int j = 1; j < kMine; ++j) mine = max(mine, group[j]);
        most = __reduce_max_sync(0xffffffffu, mine);
        const bool owner = tid == __ffs(__ballot_sync(0xffffffffu, mine == most)) - 1;
        bool gone = !owner;
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (!gone && group[j] == most) group[j] = 0, gone = true;
    }
    if (tid == 0) sh.threshold = max(most, 1u);  // (fewer groups than alternatives: whatever exists)
}

// Fewer candidates, where there are many: those that are at least the top-th largest among the maxima of 128 groups of them.
template <int kThreads>
__device__ __forceinline__ void refine(int top, Shared& sh) {
    const int tid = threadIdx.x, count = sh.candidates;
    if (count <= 2 * kMaxTop + 32) return;
    for (int g = tid; g < kGroups; g += kThreads) {
        uint64_t most = 0;
        for (int c = g; c < count; c += kGroups) most = max(most, sh.candidate[c]);
        sh.group[g] = static_cast<uint32_t>(most >> 32);
    }
    constexpr int kMine = kCandidates / kThreads;
    uint64_t mine[kMine];
#pragma unroll
    for (int c = 0; c < kMine; ++c) mine[c] = c * kThreads + tid < count ? sh.candidate[c * kThreads + tid] : 0;
    block_sync<kThreads>();
    if (tid == 0) sh.candidates = 0;
    largest_groups(top, sh);
    block_sync<kThreads>();
    const uint32_t threshold = sh.threshold;
#pragma unroll
    for (int c = 0; c < kMine; ++c)
        if (static_cast<uint32_t>(mine[c] >> 32) >= threshold) sh.candidate[atomicAdd(&sh.candidates, 1)] = mine[c];
    block_sync<kThreads>();
}

// The block's alternatives among its units [0, n) (unit 0 is unit `first` of the row), from the units' maxima, into sh.best.
template <typename T, int kThreads>
__device__ __forceinline__ void search(const Row<T>& row, int first, int n, int top, uint32_t* maxima, Shared& sh) {
    constexpr int N = Elements<T>::N;
    const int tid = threadIdx.x;
    const int per = ((n + kGroups - 1) / kGroups) | 1;  // odd: a thread's stride through shared memory meets every bank
    for (int g = tid; g < kGroups; g += kThreads) {
        uint32_t best = 0;
        for (int u = g * per; u < min(n, (g + 1) * per); ++u) best = max(best, maxima[u]);
        sh.group[g] = best;
    }
    if (tid < kMaxTop) sh.best[tid] = 0;
    if (tid == 0) sh.units = sh.candidates = 0;
    block_sync<kThreads>();
    largest_groups(top, sh);
    block_sync<kThreads>();
    const uint32_t threshold = sh.threshold;
    for (int u = tid; u < n; u += kThreads)
        if (maxima[u] >= threshold) {
            const int slot = atomicAdd(&sh.units, 1);
            if (slot < kChosen) sh.unit[slot] = u;
        }
    block_sync<kThreads>();
    const int units = sh.units;
    // (a warp alone has chosen few, but for ties; and reads its units four lanes to each, eight bytes in one load: 2048 x 1000 fp16 with five
    // alternatives 11.0 -> 9.5 us, and one masked row among them 19.7 -> 13.1.  Of more threads each reads an element: 16384 x 32768 246 us, 254 with eight bytes)
    const int enough = kThreads == 32 ? 2 * top + 8 : kChosen;
    if (units <= enough) {
        if constexpr (kThreads == 32) {
            constexpr int kPart = N / 4;
            const int lane = tid & 31;
            for (int e = tid; e - lane < units * 4; e += kThreads) {
                uint32_t key[kPart];
                const int u = e < units * 4 ? first + sh.unit[e >> 2] : 0;
                const long long i = row.first(u) + (e & 3) * kPart;
                const T* const at = row.at(u) + (e & 3) * kPart;
                const bool whole = e < units * 4 && i >= 0 && i + kPart <= row.vocab;
                uint2 v = make_uint2(0, 0);
                if (whole) v = load_global(reinterpret_cast<const uint2*>(at));
#pragma unroll
                for (int j = 0; j < kPart; ++j) {
                    const bool there = e < units * 4 && row.has(i + j);
                    key[j] = !there ? 0 : order_key(whole ? Elements<T>::of(v, j) : Elements<T>::load(at + j));
                }
                unsigned who[kPart];
                int all = 0, slot = 0;
#pragma unroll
                for (int j = 0; j < kPart; ++j) {
                    who[j] = __ballot_sync(0xffffffffu, key[j] >= threshold);
                    all += __popc(who[j]);
                }
                if (all == 0) continue;
                if (lane == 0) slot = atomicAdd(&sh.candidates, all);
                slot = __shfl_sync(0xffffffffu, slot, 0);
#pragma unroll
                for (int j = 0; j < kPart; ++j) {
                    const int mine = slot + __popc(who[j] & ((1u << lane) - 1));
                    if (key[j] >= threshold && mine < kCandidates) sh.candidate[mine] = candidate(key[j], i + j);
                    slot += __popc(who[j]);
                }
            }
        } else {
            for (int e = tid; e < units * N; e += kThreads) {
                const int u = first + sh.unit[e / N];
                const long long i = row.first(u) + e % N;
                const uint32_t k = row.has(i) ? order_key(Elements<T>::load(row.at(u) + e % N)) : 0;
                if (k >= threshold) {
                    const int slot = atomicAdd(&sh.candidates, 1);
                    if (slot < kCandidates) sh.candidate[slot] = candidate(k, i);
                }
            }
        }
    }
    block_sync<kThreads>();
    const bool listed = units <= enough && sh.candidates <= kCandidates;
    block_sync<kThreads>();
    if (listed) {
        refine<kThreads>(top, sh);
        place<kThreads>(sh.candidate, sh.candidates, top, sh.best);
    } else if (tid < 32) {
        search_units(row, first, n, per, top, maxima, sh);
    }
    block_sync<kThreads>();
}

struct ForwardParams {
    const void* logits;
    const long long* targets;
    long long rows, pitch;
    int vocab, top, cluster, share;  // share: room for maxima
    float *log_probs, *entropy, *stats, *top_log_probs;
    long long* top_indices;
};

// A row to a block, or to a cluster of blocks that take equal runs of its units and meet in the first one's shared memory.
// kFlight units of a thread are in flight: four where there are few rows, and latency counts (1 x 131072 fp32 9.4 -> 7.3 us); with two, of many rows more
// warps fit an SM (16384 x 32768 fp16 with eight alternatives 215 us, with four 231).
template <typename T, int kThreads, int kFlight>
__global__ void __launch_bounds__(kThreads == 32 ? 32 * kWarpRows : kThreads, kThreads == 32 ? 5 : 0) token_log_probs_kernel(const ForwardParams P) {
    pdl_enter();
    namespace cg = cooperative_groups;
    constexpr int kRows = kThreads == 32 ? kWarpRows : 1;
    __shared__ __align__(16) Shared all[kRows];
    extern __shared__ uint32_t all_maxima[];
    Shared& sh = all[kRows > 1 ? threadIdx.y : 0];
    uint32_t* const maxima = all_maxima + (kRows > 1 ? threadIdx.y * P.share : 0);
    const int rank = P.cluster > 1 ? static_cast<int>(blockIdx.x % P.cluster) : 0;
    const int tid = threadIdx.x;
    const long long r = kRows > 1 ? static_cast<long long>(blockIdx.x) * kRows + threadIdx.y : blockIdx.x / P.cluster;
    if (kRows > 1 && r >= P.rows) return;
    const Row<T> row(static_cast<const T*>(P.logits) + r * P.pitch, P.vocab);
    const int share = (row.units + P.cluster - 1) / P.cluster;
    const int u0 = min(row.units, rank * share), u1 = min(row.units, u0 + share);
    Running<T> run;
    auto take = [&](int u, const uint32_t (&v)[8]) {
        const float most = run.add(v);
        if (P.top) maxima[u - u0] = order_key(most);
    };
    const int f0 = max(u0, row.full0), f1 = min(u1, row.full1);
    int u = f0 + tid;
    long long target = tid == 0 ? load_index(P.targets + r) : -1;
    for (; u + (kFlight - 1) * kThreads < f1; u += kFlight * kThreads) {
        uint32_t v[kFlight][8];
#pragma unroll
        for (int e = 0; e < kFlight; ++e) load_unit(row.at(u + e * kThreads), v[e]);
#pragma unroll
        for (int e = 0; e < kFlight; ++e) take(u + e * kThreads, v[e]);
    }
    if (u < f1) {
        uint32_t v[kFlight - 1][8];
#pragma unroll
        for (int e = 0; e < kFlight - 1; ++e)
            if (u + e * kThreads < f1) load_unit(row.at(u + e * kThreads), v[e]);
#pragma unroll
        for (int e = 0; e < kFlight - 1; ++e)
            if (u + e * kThreads < f1) take(u + e * kThreads, v[e]);
    }
    // (asked for before the sums are exchanged, needed behind them)
    const float of_target = target >= 0 && target < P.vocab ? Elements<T>::load(static_cast<const T*>(P.logits) + r * P.pitch + target) : 0.f;
    // the first and the last unit, where they have gaps
    if (tid < 2) {
        const int e = tid == 0 ? 0 : row.units - 1;
        const bool broken = tid == 0 ? row.full0 == 1 : row.full1 < row.units && !(row.full0 == 1 && row.units == 1);
        if (broken && e >= u0 && e < u1) {
            uint32_t a[8];
            row.load_broken(e, a);
            take(e, a);
        }
    }
    Stats a = run.done();
    if (kThreads > 32) {
        if ((tid & 31) == 0) sh.warp[tid / 32] = a;
        __syncthreads();
        if (tid < 32) a = merge_lanes<T>(sh.warp[tid % (kThreads / 32)], kThreads / 32);
    }
    if (P.top) {
        block_sync<kThreads>();
        search<T, kThreads>(row, u0, u1 - u0, P.top, maxima, sh);
    }
    if (P.cluster > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0) sh.block = a;
        cluster.sync();
        if (rank == 0) {
            if (tid < 32) a = merge_lanes<T>(*cluster.map_shared_rank(&sh.block, tid % P.cluster), P.cluster);
            if (P.top) {
                const int count = P.cluster * P.top;
                for (int e = tid; e < count; e += kThreads) sh.candidate[e] = cluster.map_shared_rank(sh.best, e / P.top)[e % P.top];
                __syncthreads();
                place<kThreads>(sh.candidate, count, P.top, sh.best);
                __syncthreads();
            }
        }
    }
    if (rank == 0 && tid < 32) {
        const bool dead = a.m == -INFINITY, bad = !(a.m < INFINITY);  // nothing but -inf; a NaN or +inf
        const float off = below<T>(a.m);
        const float log_sum = dead ? 0.f : bad ? NAN : logf(a.s) - off * kLn2;
        if (tid < P.top) {
            const uint64_t c = sh.best[tid];
            P.top_indices[r * P.top + tid] = index_of(c);
            P.top_log_probs[r * P.top + tid] = dead ? -INFINITY : (value_of(c) - a.m) - log_sum;
        }
        if (tid == 0) {
            P.log_probs[r] = target < 0 ? 0.f : target >= P.vocab ? NAN : dead ? -INFINITY : (of_target - a.m) - log_sum;
            P.entropy[r] = dead ? 0.f : bad ? NAN : logf(a.s) - kLn2 * (a.t / a.s);
            P.stats[2 * r] = a.m;
            P.stats[2 * r + 1] = log_sum;
        }
    }
    if (P.cluster > 1) cg::this_cluster().sync();  // (the first block has read the others' shared memory)
}

struct BackwardParams {
    const void* logits;
    const long long* targets;
    const float *stats, *entropy, *d_log_probs, *d_entropy;
    void* out;
    long long rows, pitch, out_pitch;
    int vocab, blocks_per_row;
    bool together;  // rows of the logits and of the result start at the same place of a unit
};

// A block to a run of a row's units, or to several short rows (blockDim.y).
template <typename T, bool kShort>
__global__ void __launch_bounds__(256) token_log_probs_backward_kernel(const BackwardParams P) {
    pdl_enter();
    constexpr int N = Elements<T>::N;
    const long long r = kShort ? static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x / P.blocks_per_row;
    if (kShort && r >= P.rows) return;
    const int part = kShort ? 0 : static_cast<int>(blockIdx.x % P.blocks_per_row);
    const Row<T> row(static_cast<const T*>(P.logits) + r * P.pitch, P.vocab);
    T* const out = static_cast<T*>(P.out) + r * P.out_pitch;
    const float m = load_global(P.stats + 2 * r), log_sum = load_global(P.stats + 2 * r + 1);
    const long long target = load_index(P.targets + r);
    const float g = target < 0 ? 0.f : target < P.vocab ? load_global(P.d_log_probs + r) : NAN;
    const float gh = P.d_entropy ? load_global(P.d_entropy + r) : 0.f;
    const float h = P.d_entropy ? load_global(P.entropy + r) : 0.f;
    const bool dead = m == -INFINITY && log_sum == 0.f, far = extreme<T>(m);
    // With y = log2 p: d = -2^y (g + gh (y ln 2 + h)).  y = x log2 e - M - k, where M is m log2 e rounded and k what else belongs to it.
    const float M = __fmul_rn(m, kLog2e), k = fmaf(m, kLog2e, -M) + log_sum * kLog2e;
    const uint64_t l2 = pack2(kLog2e, kLog2e), m2 = pack2(-M, -M), k2 = pack2(-k, -k);
    const float slope = -gh * kLn2, level = -fmaf(gh, h, g);
    const uint64_t slope2 = pack2(slope, slope), level2 = pack2(level, level);
    const bool entropy = P.d_entropy != nullptr;
    for (int u = part * blockDim.x + threadIdx.x; u < row.units; u += (kShort ? 1 : P.blocks_per_row) * blockDim.x) {
        const bool full = u >= row.full0 && u < row.full1;
        uint32_t v[8];
        if (full) load_unit(row.at(u), v); else row.load_broken(u, v);
        uint64_t x[N / 2];
        if (!far) {
            Elements<T>::pairs(v, x);
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j)
                x[j] = pack2(max_nan((Elements<T>::get(v, 2 * j) - m) * kLog2e, -1e5f), max_nan((Elements<T>::get(v, 2 * j + 1) - m) * kLog2e, -1e5f));
        }
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            uint64_t y;
            if (far) y = add2(x[j], pack2(-log_sum * kLog2e, -log_sum * kLog2e));
            else y = add2(fma2(x[j], l2, m2), k2);
            if (sizeof(T) == 4) y = pack2(max_nan(low(y), -1e5f), max_nan(high(y), -1e5f));  // (times a gradient of any size; a row with NaN keeps it)
            const uint64_t e = pack2(power2(low(y)), power2(high(y)));
            x[j] = mul2(e, entropy ? fma2(y, slope2, level2) : level2);
        }
        const long long first = row.first(u);
        if (target >= first && target < first + N && target >= 0) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                if (target - first == 2 * j) x[j] = pack2(low(x[j]) + g, high(x[j]));
                if (target - first == 2 * j + 1) x[j] = pack2(low(x[j]), high(x[j]) + g);
            }
        }
        if (dead) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) x[j] = 0;
        }
        if (P.together && full) {
            Elements<T>::pack(x, v);
            store_unit(out + first, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (row.has(first + j)) out[first + j] = Elements<T>::round(j & 1 ? high(x[j / 2]) : low(x[j / 2]));
        }
    }
}

struct ForwardPlan {
    int threads = 0, cluster = 1, flight = 2;
    int share = 0;
    size_t smem = 0;
    bool ok = false;
};
static ForwardPlan forward_plan(long long rows, int vocab, int dtype, int top) {
    const int n = dtype == NML_F16 ? Elements<__half>::N : Elements<float>::N;
    const int units = static_cast<int>((static_cast<long long>(vocab) + 2 * n - 2) / n);  // at the worst start of a row
    ForwardPlan p;
    // A warp to a short row, four to others, eight to the longest (16384 x 32768 fp16, eight alternatives: four 215 us, eight 244; 2048 x 131072: 143 and
    // 119); these over several blocks where there are few rows.
    p.threads = units <= 128 ? 32 : units <= 4096 ? 128 : 256;
    if (units > 1024 && rows < 74) p.threads = 256;
    while (p.cluster < kMaxCluster && p.threads == 256 && ((rows * p.cluster < 148 && units > 512 * p.cluster) || (top && (units + p.cluster - 1) / p.cluster > kMaxUnits))) p.cluster *= 2;
    if (rows * p.cluster <= 148) p.flight = 4;
    p.share = (units + p.cluster - 1) / p.cluster;
    p.ok = !top || p.share <= kMaxUnits;
    p.smem = top ? sizeof(uint32_t) * p.share * (p.threads == 32 ? kWarpRows : 1) : 0;
    return p;
}
typedef void (*ForwardKernel)(const ForwardParams);
template <typename T>
static ForwardKernel forward_kernel_of(const ForwardPlan& p) {
    return p.threads == 32 ? token_log_probs_kernel<T, 32, 4> : p.threads == 128 ? token_log_probs_kernel<T, 128, 2>
           : p.flight == 4 ? token_log_probs_kernel<T, 256, 4> : token_log_probs_kernel<T, 256, 2>;
}
static ForwardKernel forward_kernel(int dtype, const ForwardPlan& p) { return dtype == NML_F16 ? forward_kernel_of<__half>(p) : forward_kernel_of<float>(p); }

static bool shape_ok(const void* logits, int dtype, long long rows, int vocab, long long pitch) {
    if (!logits || (dtype != NML_F16 && dtype != NML_F32) || rows <= 0 || vocab <= 0 || pitch < vocab) return false;
    return reinterpret_cast<uintptr_t>(logits) % (dtype == NML_F16 ? 2 : 4) == 0;
}
template <class... P>
static bool aligned(size_t to, const P*... p) {
    return (((reinterpret_cast<uintptr_t>(p) % to) == 0) && ...);
}

}  // namespace nml_logits

using namespace nml_logits;

int nml::prepare_logits_kernels() {
    for (int dtype : {NML_F32, NML_F16})
        for (int threads : {32, 128, 256})
            for (int flight : {2, 4}) {
                ForwardPlan p;
                p.threads = threads;
                p.flight = flight;
                NMLG_CUDA(cudaFuncSetAttribute(forward_kernel(dtype, p), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxUnits * 4));
            }
    cudaFuncAttributes a;
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<float, true>));
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<float, false>));
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<__half, true>));
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<__half, false>));
    return NML_OK;
}

extern "C" {

int nml_token_log_probs(const void* logits, int dtype, long long rows, int vocab, long long pitch, const long long* targets, int top,
                        float* log_probs, float* entropy, float* stats, float* top_log_probs, long long* top_indices, void* stream) {
    if (!shape_ok(logits, dtype, rows, vocab, pitch) || !targets || !log_probs || !entropy || !stats) return NML_ERR_INVALID;
    if (top < 0 || top > vocab || (top > 0 && (!top_log_probs || !top_indices))) return NML_ERR_INVALID;
    if (!aligned(4, log_probs, entropy, stats, top_log_probs) || !aligned(8, targets, top_indices)) return NML_ERR_INVALID;
    const ForwardPlan plan = forward_plan(rows, vocab, dtype, top);
    if (top > kMaxTop || !plan.ok) return NML_ERR_UNSUPPORTED;
    int* status;
    int sms;
    if (const int rc = nml::current_device(&status, &sms)) return rc;
    const ForwardParams P = {logits, targets, rows, pitch, vocab, top, plan.cluster, plan.share, log_probs, entropy, stats, top_log_probs, top_indices};
    const bool warps = plan.threads == 32;
    const long long blocks = warps ? (rows + kWarpRows - 1) / kWarpRows : rows * plan.cluster;
    if (blocks > 0x7fffffff) return NML_ERR_UNSUPPORTED;
    // (a row to a block however many there are: 16384 x 32768 fp16 188 us, 193 with 4736 blocks that take rows in turn, 199 with as many as fit the SMs)
    const int grid = static_cast<int>(blocks);
    nml::launch_with(nml::overlaps(grid, nml::kSms), plan.cluster, forward_kernel(dtype, plan), grid, warps ? dim3(32, kWarpRows) : dim3(plan.threads),
                     plan.smem,
                     static_cast<cudaStream_t>(stream), P);
    NMLG_CUDA(cudaGetLastError());
    nml::count_launches(1);
    return NML_OK;
}

int nml_token_log_probs_backward(const void* logits, int dtype, long long rows, int vocab, long long pitch, const long long* targets,
                                 const float* stats, const float* entropy, const float* d_log_probs, const float* d_entropy, void* d_logits,
                                 long long d_pitch, void* stream) {
    if (!shape_ok(logits, dtype, rows, vocab, pitch) || !shape_ok(d_logits, dtype, rows, vocab, d_pitch)) return NML_ERR_INVALID;
    if (!targets || !stats || !d_log_probs || (d_entropy && !entropy)) return NML_ERR_INVALID;
    if (!aligned(4, stats, entropy, d_log_probs, d_entropy) || !aligned(8, targets)) return NML_ERR_INVALID;
    const int size = dtype == NML_F16 ? 2 : 4, n = kUnitBytes / size;
    {  // the result: element for element where the logits are, or apart from them; and from what its row's blocks read first
        auto runs = [&](const void* p, long long count, long long length, long long step) {
            return nml::Runs{reinterpret_cast<uintptr_t>(p), count, length, step};
        };
        const nml::Runs out = runs(d_logits, rows, static_cast<long long>(vocab) * size, d_pitch * size);
        const bool in_place = d_logits == logits && (d_pitch == pitch || rows == 1);
        if (!in_place && overlap(out, runs(logits, rows, static_cast<long long>(vocab) * size, pitch * size))) return NML_ERR_INVALID;
        auto meets = [&](const void* p, long long each) { return p && overlap(out, runs(p, 1, rows * each, rows * each)); };
        if (meets(targets, 8) || meets(stats, 8) || meets(d_log_probs, 4) || meets(d_entropy, 4) || (d_entropy && meets(entropy, 4))) return NML_ERR_INVALID;
    }
    int* status;
    int sms;
    if (const int rc = nml::current_device(&status, &sms)) return rc;
    const long long units = (static_cast<long long>(vocab) + 2 * n - 2) / n;
    long long per_row = (units + 2047) / 2048;  // eight units a thread
    if (rows * per_row > 0x7fffffff) per_row = 1;
    if (rows > 0x7fffffff) return NML_ERR_UNSUPPORTED;
    const bool together = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(d_logits)) % kUnitBytes == 0 &&
                          (pitch - d_pitch) * size % kUnitBytes == 0;
    const BackwardParams P = {logits, targets, stats, entropy, d_log_probs, d_entropy, d_logits, rows, pitch, d_pitch, vocab,
                              static_cast<int>(per_row), together};
    // A power of two of threads to a row, up to two units each where it is short, 256 to a block.
    int threads = 8;
    while (threads < 256 && 2 * threads < units) threads *= 2;
    const dim3 block(threads, 256 / threads);
    const long long blocks = (rows + block.y - 1) / block.y * per_row;
    nml::launch(dtype == NML_F16 ? (threads < 256 ? token_log_probs_backward_kernel<__half, true> : token_log_probs_backward_kernel<__half, false>)
                                 : (threads < 256 ? token_log_probs_backward_kernel<float, true> : token_log_probs_backward_kernel<float, false>),
                static_cast<unsigned>(blocks), block, 0, static_cast<cudaStream_t>(stream), P);
    NMLG_CUDA(cudaGetLastError());
    nml::count_launches(1);
    return NML_OK;
}

}  // extern "C"
