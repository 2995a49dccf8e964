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
// Units.  A row is read in units of 32 bytes (one load of 256 bits) that start on 32-byte boundaries of memory, so a row of an
// odd vocabulary, which starts anywhere, is read like any other; its first and last unit are taken element by element.
//
// Alternatives.  The pass also notes the largest logit of every unit.  The `top` largest elements of a row lie in the `top`
// units with the largest maxima (a unit that holds one of them has a maximum no element outside those units beats; ties go to the lower index on
// both levels, as units are contiguous), so those few units are read again and searched; the row is not.
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

constexpr int kMaxTop = 32;          // a lane for each selected unit
constexpr int kUnitBytes = 32;
constexpr int kGroups = 256;         // of units, for the search: eight to a lane
constexpr int kMaxUnits = 63 * kGroups;  // of one block's share of a row: its maxima take 63 KB
constexpr int kMaxCluster = 8;

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

template <typename T>
struct Elements;
template <>
struct Elements<float> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint32_t (&v)[8], float (&x)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = __uint_as_float(v[j]);
    }
    static __device__ __forceinline__ void pack(const float (&x)[N], uint32_t (&v)[8]) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = __float_as_uint(x[j]);
    }
    static __device__ __forceinline__ float load(const float* p) { return load_global(p); }
    static __device__ __forceinline__ float round(float x) { return x; }
};
template <>
struct Elements<__half> {
    static constexpr int N = 16;
    static __device__ __forceinline__ void unpack(const uint32_t (&v)[8], float (&x)[N]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[j]));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void pack(const float (&x)[N], uint32_t (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<__half2*>(&v[j]) = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
    }
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(load_global(p)); }
    static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};

// Floats in the order of unsigned integers (-0 and 0 are one value; NaN above everything).  0 is below every float: "none".
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A row as units: unit u holds the elements u * N - lead ... of which those in [0, vocab) exist.
template <typename T>
struct Row {
    const T* base;  // of unit 0: at or before the row's first element, on a 32-byte boundary
    int lead, vocab, units;
    __device__ __forceinline__ Row(const T* row, int vocab_) {
        lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) & (kUnitBytes - 1)) / sizeof(T));
        base = row - lead;
        vocab = vocab_;
        units = static_cast<int>((static_cast<long long>(lead) + vocab + Elements<T>::N - 1) / Elements<T>::N);
    }
    __device__ __forceinline__ bool full(int u) const {
        return (u > 0 || lead == 0) && (u + 1 < units || (lead + static_cast<long long>(vocab)) % Elements<T>::N == 0);
    }
    // The unit's elements; `none` where there is none.
    __device__ __forceinline__ void load(int u, float none, float (&x)[Elements<T>::N]) const {
        const T* p = base + static_cast<long long>(u) * Elements<T>::N;
        if (full(u)) {
            uint32_t v[8];
            load_unit(p, v);
            Elements<T>::unpack(v, x);
        } else {
#pragma unroll
            for (int j = 0; j < Elements<T>::N; ++j) {
                const long long i = static_cast<long long>(u) * Elements<T>::N + j - lead;
                x[j] = i >= 0 && i < vocab ? Elements<T>::load(p + j) : none;
            }
        }
    }
};

// Running statistics: the maximum, sum e^(x - m) and sum (x - m) e^(x - m).  While everything is -inf, m is -inf and the sums are 0.
struct Stats {
    float m, s, t;
};
constexpr float kLog2e = 1.4426950408889634f;
// e^d underflows to 0 well above this; it keeps (x - m) e^(x - m) at 0 where x is -inf.
constexpr float kLowest = -200.f;

__device__ __forceinline__ float exp_of(float d) { return exp2f(d * kLog2e); }

// The same statistics against a larger maximum.
__device__ __forceinline__ void raise(Stats& a, float m) {
    if (a.m < m) {
        if (a.s != 0.f) {  // (so m is finite; a sum that is NaN stays it)
            const float d = a.m - m, f = exp_of(d);
            a.t = (a.t + fmaxf(d, kLowest) * a.s) * f;
            a.s *= f;
        }
        a.m = m;
    }
}
__device__ __forceinline__ void merge(Stats& a, Stats b) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m);
    raise(b, m);
    a.s += b.s;
    a.t += b.t;
}

template <typename T>
__device__ __forceinline__ float add_unit(Stats& a, const float (&x)[Elements<T>::N]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < Elements<T>::N; ++j) m = fmaxf(m, x[j]);
    raise(a, m);
    const float ref = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int j = 0; j < Elements<T>::N; ++j) {
        const float d = x[j] - ref, e = exp_of(d);
        a.s += e;
        a.t += fmaxf(d, kLowest) * e;
    }
    return m;
}

__device__ __forceinline__ Stats shuffle(const Stats& a, int o) {
    return {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
}

// One block's part of the search, and a cluster's exchange.
struct Shared {
    Stats warp[8], block;
    uint32_t group[kGroups];
    int chosen[kMaxTop];
    uint32_t key[kMaxTop];   // the block's alternatives, in order
    int index[kMaxTop];
};

template <int kThreads>
__device__ __forceinline__ void block_sync() {
    if (kThreads == 32) __syncwarp(); else __syncthreads();
}

// The `top` largest of up to 32 x 8 candidates in registers, by value, then by index; lane r receives the r-th.
template <int N>
__device__ __forceinline__ void select(uint32_t (&key)[N], const int (&index)[N], int top, uint32_t& out_key, int& out_index) {
    const int lane = threadIdx.x & 31;
    out_key = 0;
    out_index = 0;
    for (int r = 0; r < top; ++r) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) best = max(best, key[j]);
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        uint32_t first = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (key[j] == most) first = min(first, static_cast<uint32_t>(index[j]));
        const uint32_t who = __reduce_min_sync(0xffffffffu, first);
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (key[j] == most && static_cast<uint32_t>(index[j]) == who) key[j] = 0;
        if (lane == r) {
            out_key = most;
            out_index = static_cast<int>(who);
        }
    }
}

// The block's alternatives among its units [0, n) (unit 0 is unit `first` of the row), from the units' maxima, into sh.key and sh.index.
template <typename T, int kThreads>
__device__ __forceinline__ void search(const Row<T>& row, int first, int n, int top, uint32_t* maxima, Shared& sh) {
    const int per = ((n + kGroups - 1) / kGroups) | 1;  // odd: a thread's stride through shared memory meets every bank
    for (int g = threadIdx.x; g < kGroups; g += kThreads) {
        uint32_t best = 0;
        for (int i = g * per; i < min(n, (g + 1) * per); ++i) best = max(best, maxima[i]);
        sh.group[g] = best;
    }
    block_sync<kThreads>();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        uint32_t group[kGroups / 32];
#pragma unroll
        for (int j = 0; j < kGroups / 32; ++j) group[j] = sh.group[lane * (kGroups / 32) + j];
        int found = 0;
        for (; found < top; ++found) {
            uint32_t best = 0;
            int at = 0;
#pragma unroll
            for (int j = kGroups / 32 - 1; j >= 0; --j)
                if (group[j] >= best) best = group[j], at = j;
            const uint32_t most = __reduce_max_sync(0xffffffffu, best);
            if (most == 0) break;  // fewer units than alternatives
            const int owner = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
            const int g = __shfl_sync(0xffffffffu, lane * (kGroups / 32) + at, owner);
            // its first unit with that maximum, and its maximum without that unit
            const int lo = g * per, a = lo + lane, b = a + 32;
            const bool has_a = lane < per && a < n, has_b = lane + 32 < per && b < n;
            const uint32_t va = has_a ? maxima[a] : 0, vb = has_b ? maxima[b] : 0;
            const unsigned in_a = __ballot_sync(0xffffffffu, has_a && va == most), in_b = __ballot_sync(0xffffffffu, has_b && vb == most);
            const int unit = lo + (in_a ? __ffs(in_a) - 1 : 32 + __ffs(in_b) - 1);
            const uint32_t rest = __reduce_max_sync(0xffffffffu, max(a == unit ? 0u : va, b == unit ? 0u : vb));
            if (lane == 0) {
                maxima[unit] = 0;
                sh.chosen[found] = unit;
            }
            if (lane == owner) {
#pragma unroll
                for (int j = 0; j < kGroups / 32; ++j)
                    if (j == at) group[j] = rest;
            }
            __syncwarp();
        }
        // a lane to a unit; the elements are compared by value, then index
        uint32_t key[Elements<T>::N];
        int index[Elements<T>::N];
#pragma unroll
        for (int j = 0; j < Elements<T>::N; ++j) key[j] = 0, index[j] = 0;
        if (lane < found) {
            const int u = first + sh.chosen[lane];
            float x[Elements<T>::N];
            row.load(u, 0.f, x);
#pragma unroll
            for (int j = 0; j < Elements<T>::N; ++j) {
                const long long i = static_cast<long long>(u) * Elements<T>::N + j - row.lead;
                index[j] = static_cast<int>(i);
                key[j] = i >= 0 && i < row.vocab ? order_key(x[j]) : 0;
            }
        }
        uint32_t k;
        int i;
        select(key, index, top, k, i);
        if (lane < top) {
            sh.key[lane] = k;
            sh.index[lane] = i;
        }
        __syncwarp();
    }
}

struct ForwardParams {
    const void* logits;
    const long long* targets;
    long long rows, pitch;
    int vocab, top, cluster;
    float *log_probs, *entropy, *stats, *top_log_probs;
    long long* top_indices;
};

// A row to a block, or to a cluster of blocks that take equal runs of its units and meet in the first one's shared memory.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_log_probs_kernel(const ForwardParams P) {
    pdl_enter();
    namespace cg = cooperative_groups;
    __shared__ Shared sh;
    extern __shared__ uint32_t maxima[];
    constexpr int N = Elements<T>::N;
    const int rank = P.cluster > 1 ? static_cast<int>(blockIdx.x % P.cluster) : 0;
    const int tid = threadIdx.x;
    for (long long r = blockIdx.x / P.cluster; r < P.rows; r += gridDim.x / P.cluster) {
        const Row<T> row(static_cast<const T*>(P.logits) + r * P.pitch, P.vocab);
        const int share = (row.units + P.cluster - 1) / P.cluster;
        const int u0 = min(row.units, rank * share), u1 = min(row.units, u0 + share);
        Stats a = {-INFINITY, 0.f, 0.f};
        for (int u = u0 + tid; u < u1; u += kThreads) {
            float x[N];
            row.load(u, -INFINITY, x);
            const float m = add_unit<T>(a, x);
            if (P.top) {
                float best = m;  // (a maximum passes over NaN)
#pragma unroll
                for (int j = 0; j < N; ++j) best = x[j] != x[j] ? x[j] : best;
                maxima[u - u0] = order_key(best);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o /= 2) merge(a, shuffle(a, o));
        if (kThreads > 32) {
            if ((tid & 31) == 0) sh.warp[tid / 32] = a;
            __syncthreads();
            a = sh.warp[0];
#pragma unroll
            for (int w = 1; w < kThreads / 32; ++w) merge(a, sh.warp[w]);
        }
        if (P.top) {
            block_sync<kThreads>();
            search<T, kThreads>(row, u0, u1 - u0, P.top, maxima, sh);
        }
        uint32_t key = 0;
        int index = 0;
        if (P.cluster > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (tid == 0) sh.block = a;
            cluster.sync();
            if (rank == 0 && tid < 32) {
                for (int c = 1; c < P.cluster; ++c) merge(a, *cluster.map_shared_rank(&sh.block, c));
                if (P.top) {
                    uint32_t keys[kMaxCluster];
                    int indices[kMaxCluster];
#pragma unroll
                    for (int c = 0; c < kMaxCluster; ++c) {
                        keys[c] = c < P.cluster && tid < P.top ? cluster.map_shared_rank(sh.key, c)[tid] : 0;
                        indices[c] = c < P.cluster && tid < P.top ? cluster.map_shared_rank(sh.index, c)[tid] : 0;
                    }
                    select(keys, indices, P.top, key, index);
                }
            }
        } else if (P.top && tid < P.top) {
            key = sh.key[tid];
            index = sh.index[tid];
        }
        if (rank == 0 && tid < 32) {
            const bool dead = a.s == 0.f;  // nothing but -inf
            const float log_sum = dead ? 0.f : logf(a.s);
            if (tid < P.top) {
                P.top_indices[r * P.top + tid] = index;
                P.top_log_probs[r * P.top + tid] = dead ? -INFINITY : (key_value(key) - a.m) - log_sum;
            }
            if (tid == 0) {
                const long long target = load_index(P.targets + r);
                float lp = 0.f;
                if (target >= P.vocab) {
                    lp = NAN;
                } else if (target >= 0) {
                    const float x = Elements<T>::load(static_cast<const T*>(P.logits) + r * P.pitch + target);
                    lp = dead ? -INFINITY : (x - a.m) - log_sum;
                }
                P.log_probs[r] = lp;
                P.entropy[r] = dead ? 0.f : log_sum - a.t / a.s;
                P.stats[2 * r] = a.m;
                P.stats[2 * r + 1] = log_sum;
            }
        }
        if (P.cluster > 1) cg::this_cluster().sync(); else block_sync<kThreads>();
    }
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

// A block to a run of a row's units.
template <typename T>
__global__ void __launch_bounds__(256) token_log_probs_backward_kernel(const BackwardParams P) {
    pdl_enter();
    constexpr int N = Elements<T>::N;
    const long long r = blockIdx.x / P.blocks_per_row;
    const int part = static_cast<int>(blockIdx.x % P.blocks_per_row);
    const Row<T> row(static_cast<const T*>(P.logits) + r * P.pitch, P.vocab);
    T* const out = static_cast<T*>(P.out) + r * P.out_pitch;
    const float m = load_global(P.stats + 2 * r), log_sum = load_global(P.stats + 2 * r + 1);
    const long long target = load_index(P.targets + r);
    const float g = target < 0 ? 0.f : target < P.vocab ? load_global(P.d_log_probs + r) : NAN;
    const float gh = P.d_entropy ? load_global(P.d_entropy + r) : 0.f;
    const float h = P.d_entropy ? load_global(P.entropy + r) : 0.f;
    const bool dead = m == -INFINITY && log_sum == 0.f;
    for (int u = part * blockDim.x + threadIdx.x; u < row.units; u += P.blocks_per_row * blockDim.x) {
        float x[N];
        row.load(u, 0.f, x);
        const long long first = static_cast<long long>(u) * N - row.lead;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float lp = (x[j] - m) - log_sum, p = exp_of(lp);
            float d = -p * (g + gh * (fmaxf(lp, kLowest) + h));
            if (first + j == target) d += g;
            x[j] = dead ? 0.f : d;
        }
        if (P.together && row.full(u)) {
            uint32_t v[8];
            Elements<T>::pack(x, v);
            store_unit(out + first, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (first + j >= 0 && first + j < P.vocab) out[first + j] = Elements<T>::round(x[j]);
        }
    }
}

struct ForwardPlan {
    int threads = 0, cluster = 1;
    size_t smem = 0;
    bool ok = false;
};
static ForwardPlan forward_plan(long long rows, int vocab, int dtype, int top) {
    const int n = dtype == NML_F16 ? Elements<__half>::N : Elements<float>::N;
    const int units = static_cast<int>((static_cast<long long>(vocab) + 2 * n - 2) / n);  // at the worst start of a row
    ForwardPlan p;
    p.threads = units <= 128 ? 32 : units <= 1024 ? 128 : 256;
    while (p.cluster < kMaxCluster && p.threads == 256 && (rows * p.cluster < 148 || (top && (units + p.cluster - 1) / p.cluster > kMaxUnits))) p.cluster *= 2;
    const int share = (units + p.cluster - 1) / p.cluster;
    p.ok = !top || share <= kMaxUnits;
    p.smem = top ? sizeof(uint32_t) * static_cast<size_t>(share) : 0;
    return p;
}
typedef void (*ForwardKernel)(const ForwardParams);
static ForwardKernel forward_kernel(int dtype, int threads) {
    if (dtype == NML_F16) return threads == 32 ? token_log_probs_kernel<__half, 32> : threads == 128 ? token_log_probs_kernel<__half, 128> : token_log_probs_kernel<__half, 256>;
    return threads == 32 ? token_log_probs_kernel<float, 32> : threads == 128 ? token_log_probs_kernel<float, 128> : token_log_probs_kernel<float, 256>;
}

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
            NMLG_CUDA(cudaFuncSetAttribute(forward_kernel(dtype, threads), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxUnits * 4));
    cudaFuncAttributes a;
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<float>));
    NMLG_CUDA(cudaFuncGetAttributes(&a, token_log_probs_backward_kernel<__half>));
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
    const ForwardParams P = {logits, targets, rows, pitch, vocab, top, plan.cluster, log_probs, entropy, stats, top_log_probs, top_indices};
    const long long blocks = rows * plan.cluster, most = static_cast<long long>(sms) * 32 / plan.cluster * plan.cluster;
    const int grid = static_cast<int>(blocks < most ? blocks : most);
    nml::launch_with(nml::overlaps(grid, nml::kSms), plan.cluster, forward_kernel(dtype, plan.threads), grid, plan.threads, plan.smem,
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
    int* status;
    int sms;
    if (const int rc = nml::current_device(&status, &sms)) return rc;
    const int size = dtype == NML_F16 ? 2 : 4, n = kUnitBytes / size;
    const long long units = (static_cast<long long>(vocab) + 2 * n - 2) / n;
    long long per_row = (units + 1023) / 1024;  // four units a thread
    if (rows * per_row > 0x7fffffff) per_row = 1;
    if (rows > 0x7fffffff) return NML_ERR_UNSUPPORTED;
    const bool together = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(d_logits)) % kUnitBytes == 0 &&
                          (pitch - d_pitch) * size % kUnitBytes == 0;
    const BackwardParams P = {logits, targets, stats, entropy, d_log_probs, d_entropy, d_logits, rows, pitch, d_pitch, vocab,
                              static_cast<int>(per_row), together};
    const int threads = units >= 256 ? 256 : static_cast<int>((units + 31) / 32 * 32);
    nml::launch(dtype == NML_F16 ? token_log_probs_backward_kernel<__half> : token_log_probs_backward_kernel<float>,
                static_cast<unsigned>(rows * per_row), threads, 0, static_cast<cudaStream_t>(stream), P);
    NMLG_CUDA(cudaGetLastError());
    nml::count_launches(1);
    return NML_OK;
}

}  // extern "C"
