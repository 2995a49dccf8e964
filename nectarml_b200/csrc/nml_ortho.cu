// Orthogonalised updates: a few steps of the iteration
//
//   X <- (a I + b A + c A^2) X,  A = X X^T,  starting at G / (|G| + eps)  (Frobenius norm),
//
// which drive the singular values of G towards 1 and keep its singular vectors, and the optimizer step that applies such an update
// to every matrix of a model (momentum, orthogonalisation, weight decay, fp16 copy).  The reference's optimizers
// (nectarml/optim/sgd.py:60-90) have no such update; this stands beside nml_sgd_momentum_step.
//
// A group of matrices is worked on at once, each turned so that it is wide: X is m x n with m <= n.  A step is three products, each one
// launch for the whole group:
//   gram     A = X X^T         symmetric, the blocks on and below the diagonal; stores A and P = b I + c A
//   square   U = a I + P A     symmetric too (polynomials of A commute)
//   update   X = U X           (the last one writes the result, or the parameters, in the caller's layout)
//
// Operands are fp16.  |X| <= 1 bounds every element of every matrix here, so powers of two chosen on the host put all of them
// into fp16's range, which needs no look at the data.
//   "3xf16" (fp32 results): every operand is a high and a low half, 22 bits, and a product is the three that matter, in fp32
//           accumulators: an error of about 2^-22 of the largest element a product, below that of fp32 products by FMA.
//   "f16"   one product.  What may not be rounded to 11 bits is X itself where it is carried from step to step: noise in directions whose singular
//           value is small grows by `a` a step (3.4^5 = 490), the signal in the others does not.  So X keeps its low half, and the
//           update adds a I times it: one more K block a tile.  (Errors of the result against 64 bits at gradients of 32 strong
//           directions, 512 x 512: 1.0e-3; with X rounded 5.9e-3; all of U X in two products 1.2e-3.)
//
// Storage.  Every matrix between the products lies in blocks of 128 x 128, a block as two halves of 64 columns, each 128
// rows of 128 bytes in the 128-byte swizzle that tcgen05.mma reads: a tile of an operand is contiguous, an untiled bulk copy brings it, no
// tensor map is needed and ragged sizes are zeros in the blocks.  Such a half serves as K-major (its rows are the M or
// N index) and as MN-major operand (its columns are), so X is read both ways, and a block of a symmetric matrix
// stands for its mirror image too.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "../../include/nectarml_b200.h"
#include "nml_host.cuh"
#include "nml_launch.cuh"
#include "nml_ptx.cuh"

namespace nml_ortho {

using nml::load_global;
using nml::pdl_enter;

#define NMLO_CUDA(expr)                                                             \
    do {                                                                            \
        const cudaError_t e_ = (expr);                                              \
        if (e_ != cudaSuccess) return nml::cuda_failed(static_cast<int>(e_), #expr); \
    } while (0)

constexpr int kGroup = 128;            // matrices of one run of launches
constexpr int kMaxSteps = 32;
constexpr int kBlock = 128;            // rows and columns of a block
constexpr uint32_t kHalf = 16384;      // bytes of one half of a block
constexpr uint32_t kPiece = 8192;      // of one copy: 64 rows of a half
constexpr uint32_t kPlane = 2 * kHalf; // of a block
constexpr int kSumElements = 8192;     // of a block of the sum of squares

// Symmetric matrices of a step, as buffers of the workspace: A, P, and U where every step has its own; T = U A, a second U and two Q (see
// Polynomial) where steps are chained.
enum { kGram = 0, kPoly = 1, kUpdate = 2, kUpdate2 = 3, kT = 4, kQ = 5, kQ2 = 6 };

// One matrix of a group as the caller has it, turned wide: element (i, j), i < m <= n, is at in + i * in_i + j * in_j.
struct Source {
    const void* in;       // the matrix, or the gradient of a parameter
    void* out;            // the result, or the parameter
    float* momentum;      // (optimizer step)
    __half* half;         // (optimizer step) fp16 copy of the parameter
    long long in_i, in_j, out_i, out_j;
    int m, n;
    float scale;          // (optimizer step) of the update
};
// and as the launches after the first find it in the workspace.
struct alignas(16) Work {
    Source s;
    uint32_t x[2], sym;                 // first blocks of X's two copies and of the symmetric matrices, in blocks of two planes
    int mb, nb;                         // blocks along m and n
    int first_sum, sums;                // its partial sums of squares
    int first_half, first_gram, first_update;  // its halves of X, tiles of the symmetric products, tiles of the update
    int wide;                           // blocks of n to a tile of the update: 1 or 2
    float sx;                           // X is stored times this
};
template <int N>
struct Group {
    Work w[N];
};

struct Common {
    const Work* table;
    const double* sums;
    uint8_t* blocks;
    const int* skip;  // the optimizer step's: do nothing where this is set
    int count;
};

// Optimizer step: u = g + momentum * v (or v) with g = grad * inv_scale and v the new momentum.
struct Momentum {
    float inv_scale, momentum;
    bool on, nesterov;
};

__device__ __forceinline__ Work load_work(const Work* p) {
    Work w;
    uint4* to = reinterpret_cast<uint4*>(&w);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(Work) / 16); ++k) to[k] = load_global(reinterpret_cast<const uint4*>(p) + k);
    return w;
}
__device__ __forceinline__ bool skipped(const int* skip) { return skip && load_global(skip) != 0; }

__device__ __forceinline__ double load_double(const double* p) {
    double v;
    asm volatile("ld.global.f64 %0, [%1];" : "=d"(v) : "l"(__cvta_generic_to_global(p)));
    return v;
}

// The matrix whose range [first, next one's first) holds k.
template <int N>
__device__ __forceinline__ int owner_of(const int (&first)[N], int count, int k) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first[mid] <= k) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float load_as_float(const T* p) { return static_cast<float>(load_global(p)); }
template <>
__device__ __forceinline__ float load_as_float<__half>(const __half* p) { return __half2float(load_global(p)); }

// ---------------------------------------------------------------- sum of squares --
// Partial sums of squares in double, kSumElements elements a block, in memory order; the optimizer step's momentum on the way.
// The first block leaves the group's table in the workspace.
template <int N, typename T>
__global__ void __launch_bounds__(256) ortho_sums_kernel(const __grid_constant__ Group<N> group, int count, Momentum mo, Work* table,
                                                         double* sums, const int* skip) {
    pdl_enter();
    __shared__ double part[8];
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < count; i += blockDim.x) table[i] = group.w[i];
    if (skipped(skip)) return;
    int k = 0;
    {
        int lo = 0, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (group.w[mid].first_sum <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
        }
        k = lo;
    }
    const Source& s = group.w[k].s;
    const bool turned = s.in_i == 1 && s.in_j != 1;  // memory runs along i
    const unsigned inner = turned ? s.m : s.n;
    const long long pitch = turned ? s.in_j : s.in_i;
    const long long total = static_cast<long long>(s.m) * s.n;
    const long long first = static_cast<long long>(blockIdx.x - group.w[k].first_sum) * kSumElements;
    const long long last = min(total, first + kSumElements);
    const T* in = static_cast<const T*>(s.in);
    double sum = 0.0;
#pragma unroll 4
    for (long long e = first + threadIdx.x; e < last; e += 256) {
        const long long outer = e / inner;
        float v = load_as_float(in + outer * pitch + (e - outer * inner));
        if (mo.on) {
            v *= mo.inv_scale;
            const float b = mo.momentum * load_global(s.momentum + e) + v;  // (dense, as the parameter)
            s.momentum[e] = b;
            v = mo.nesterov ? v + mo.momentum * b : b;
        }
        sum += static_cast<double>(v) * static_cast<double>(v);
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += part[w];
        sums[blockIdx.x] = sum;
    }
}

// ---------------------------------------------------------------- blocks --
__device__ __forceinline__ uint8_t* block_at(uint8_t* blocks, uint32_t first, int index) {
    return blocks + (static_cast<size_t>(first) + index) * (2 * kPlane);
}
// A block on or below the diagonal of a symmetric matrix.
__device__ __forceinline__ int lower(int i, int j) { return i * (i + 1) / 2 + j; }

// High and low half of a value.
__device__ __forceinline__ void split(float v, __half& h, __half& l) {
    h = __float2half_rn(v);
    l = __float2half_rn(v - __half2float(h));
}
// Sixteen adjacent columns (two 16-byte chunks, c the first) of a row of a half, in its swizzle: one 32-byte store a plane.
template <bool kLow>
__device__ __forceinline__ void store16(uint8_t* half, int row, int c, const float (&v)[16]) {
    uint32_t h[8], l[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        __half h0, l0, h1, l1;
        split(v[2 * q], h0, l0);
        split(v[2 * q + 1], h1, l1);
        __half2 a = __halves2half2(h0, h1), b = __halves2half2(l0, l1);
        h[q] = *reinterpret_cast<uint32_t*>(&a);
        l[q] = *reinterpret_cast<uint32_t*>(&b);
    }
    // chunk c lies at c ^ (row & 7): the pair is 32-byte aligned, in turned order in odd rows
    const bool odd = row & 1;
    uint8_t* p = half + row * 128 + (((c ^ (row & 7)) & ~1) << 4);
    auto put = [&](uint8_t* at, const uint32_t (&w)[8]) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(at)), "r"(odd ? w[4] : w[0]),
                     "r"(odd ? w[5] : w[1]), "r"(odd ? w[6] : w[2]), "r"(odd ? w[7] : w[3]), "r"(odd ? w[0] : w[4]), "r"(odd ? w[1] : w[5]),
                     "r"(odd ? w[2] : w[6]), "r"(odd ? w[3] : w[7])
                     : "memory");
    };
    put(p, h);
    if (kLow) put(p + kPlane, l);
}

// ---------------------------------------------------------------- first iterate --
// One half (128 x 64) of X to a block: the matrix over its norm, in two planes, zeros beyond its edges.  The blocks behind write the
// identity blocks of "f16": a_k I for every step.
struct PackParams {
    Common c;
    Momentum mo;
    float eps;
    int halves;
    uint32_t identity;  // first block
    float diagonal[kMaxSteps];
};
template <typename T>
__global__ void __launch_bounds__(256) ortho_pack_kernel(const __grid_constant__ PackParams P) {
    pdl_enter();
    if (skipped(P.c.skip)) return;
    __shared__ float tile[64][129];
    __shared__ double part[8];
    __shared__ int first[kGroup];
    const int tid = threadIdx.x;
    if (static_cast<int>(blockIdx.x) >= P.halves) {
        const int k = blockIdx.x - P.halves, half = k & 1;
        for (int o = tid; o < 128 * 4; o += 256) {
            float v[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = half * 64 + (o & 3) * 16 + q == o / 4 ? P.diagonal[k / 2] : 0.f;
            store16<true>(block_at(P.c.blocks, P.identity, k / 2) + half * kHalf, o / 4, (o & 3) * 2, v);
        }
        return;
    }
    for (int i = tid; i < P.c.count; i += 256) first[i] = load_global(&P.c.table[i].first_half);
    __syncthreads();
    const int k = owner_of(first, P.c.count, blockIdx.x);
    const Work w = load_work(P.c.table + k);
    const Source& s = w.s;
    // the norm, from the partial sums in a fixed order
    double sum = 0.0;
    for (int i = tid; i < w.sums; i += 256) sum += load_double(P.c.sums + w.first_sum + i);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) part[tid / 32] = sum;
    __syncthreads();
    sum = part[0];
#pragma unroll
    for (int q = 1; q < 8; ++q) sum += part[q];
    const double norm = sqrt(sum) + static_cast<double>(P.eps);
    const double inv = norm == 0.0 ? 0.0 : static_cast<double>(w.sx) / norm;  // (zeros stay zeros without an eps too)
    const int half = blockIdx.x - first[k], i0 = half / (2 * w.nb) * kBlock, j0 = half % (2 * w.nb) * 64;
    const T* in = static_cast<const T*>(s.in);
    auto value = [&](int i, int j) -> float {
        if (i >= s.m || j >= s.n) return 0.f;
        float v = load_as_float(in + i * s.in_i + j * s.in_j);
        if (P.mo.on) {
            v *= P.mo.inv_scale;
            const float b = load_global(s.momentum + i * s.in_i + j * s.in_j);
            v = P.mo.nesterov ? v + P.mo.momentum * b : b;
        }
        return static_cast<float>(static_cast<double>(v) * inv);
    };
    if (s.in_i == 1 && s.in_j != 1)
        for (int e = tid; e < 128 * 64; e += 256) tile[e >> 7][e & 127] = value(i0 + (e & 127), j0 + (e >> 7));
    else
        for (int e = tid; e < 128 * 64; e += 256) tile[e & 63][e >> 6] = value(i0 + (e >> 6), j0 + (e & 63));
    __syncthreads();
    uint8_t* const out = block_at(P.c.blocks, w.x[0], half / 2) + (half & 1) * kHalf;
    for (int o = tid; o < 128 * 4; o += 256) {
        const int row = o & 127, c = o >> 7;
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = tile[c * 16 + q][row];
        store16<true>(out, row, c * 2, v);
    }
}

// ---------------------------------------------------------------- products --
__device__ __forceinline__ long long load_wide(const long long* p) {
    long long v;
    asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(__cvta_generic_to_global(p)));
    return v;
}
// Sixteen results of a row, of which `count` exist, to places `step` apart; in 16-byte vectors where they lie densely.
__device__ __forceinline__ bool dense16(const void* p, long long step, int count) { return step == 1 && count >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__device__ __forceinline__ void write16(float* p, long long step, int count, const float (&v)[16]) {
    if (dense16(p, step, count)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) reinterpret_cast<float4*>(p)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    } else {
#pragma unroll
        for (int q = 0; q < 16; ++q, p += step)
            if (q < count) *p = v[q];
    }
}
__device__ __forceinline__ void write16(__half* p, long long step, int count, const float (&v)[16]) {
    if (dense16(p, step, count)) {
        uint32_t h[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            __half2 t = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
            h[q] = *reinterpret_cast<uint32_t*>(&t);
        }
        reinterpret_cast<uint4*>(p)[0] = make_uint4(h[0], h[1], h[2], h[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(h[4], h[5], h[6], h[7]);
    } else {
#pragma unroll
        for (int q = 0; q < 16; ++q, p += step)
            if (q < count) *p = __float2half_rn(v[q]);
    }
}
// The same for parameters: p = p keep - rate v, and their fp16 copy.
__device__ __forceinline__ void apply16(float* p, __half* half, long long step, int count, float (&v)[16], float keep, float rate) {
    if (dense16(p, step, count)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 w = load_global(reinterpret_cast<const float4*>(p) + q);
            v[4 * q] = w.x * keep - rate * v[4 * q];
            v[4 * q + 1] = w.y * keep - rate * v[4 * q + 1];
            v[4 * q + 2] = w.z * keep - rate * v[4 * q + 2];
            v[4 * q + 3] = w.w * keep - rate * v[4 * q + 3];
        }
    } else {
        const float* r = p;
#pragma unroll
        for (int q = 0; q < 16; ++q, r += step)
            if (q < count) v[q] = load_global(r) * keep - rate * v[q];
    }
    write16(p, step, count, v);
    if (half) write16(half, step, count, v);
}

// What a product's epilogue makes of the accumulators D.
enum {
    POLY = 0,    // symmetric: A = D, and P = b I + c A beside it
    PLAIN = 1,   // symmetric: D + d1 I
    ITERATE = 2, // X
    RESULT = 3   // X in the caller's layout, or the parameters' update
};
struct Symmetric {  // buffers of one symmetric product
    int left, right, out;
    float f0, d1;   // stored: D f0 (+ d1 on the diagonal)
};
struct ProductParams {
    Common c;
    int* err;
    int tiles, stages, from;   // from: which copy of X is read
    bool gram;                 // POLY of X X^T; else the jobs' operands
    Symmetric job[2];          // the tiles of a second one follow those of the first
    int jobs;
    float f1, d1;              // POLY: P = D f1 + d1 I
    float f0;                  // ITERATE, RESULT
    int left;                  // ITERATE, RESULT: the symmetric factor
    uint32_t identity;         // "f16": block of this step's a I
    int out_half;              // RESULT is fp16
    bool apply;                // RESULT goes into parameters: p = p keep - rate scale result
    float keep, rate;
};

constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr int kStageBytes = 196608;  // of the ring, at most
constexpr int kMaxStages = 6;
constexpr size_t kProductSmem = kStageBytes + 1024;
// The tensor core truncates where it adds to an accumulator: about 2^-24 of the sum for each instruction, all to one side (measured: 2.5 x 2^-24 of a
// sum of positive products over K = 64, 98 over 1024).  In three products over K = 8192 that was 7e-5 of the result.  So with two halves the epilogue
// warps take the accumulators of every K slice of 64 and add them in registers, rounded to nearest, while the next slice goes to the other
// accumulators; and within a slice the mixed products come first, while the sums are 2^11 times smaller: four additions count.
// (One product of halves, of 2^-12, does not need it.)

// What a tile of a product is made of.
struct Tile {
    int k;           // matrix of the group
    int i, j;        // its block row; its (first) block column
    int job;
    int groups;      // 64-column groups of it
    int slices;      // of 64 along K
    int extra;       // "f16" update: slices of a I times X's low half behind them
};
struct Info {        // of a matrix, in shared memory
    int m, n, nb, wide;
    uint32_t x[2], sym;
    float sx;
};

template <int kPlanes, int kKind>
__global__ void __launch_bounds__(kThreads, 1) ortho_product_kernel(const __grid_constant__ ProductParams P) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], tfull_bar[2], tempty_bar[2], drain_bar;
    __shared__ __align__(8) int abort_state[4];
    __shared__ uint32_t tmem_base;
    __shared__ int first[kGroup];
    __shared__ Info info[kGroup];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    volatile int* const abort_flag = abort_state;
    constexpr bool kWide = kKind >= ITERATE;
    constexpr uint32_t b_bytes = kWide ? 2 * kHalf : kHalf;  // a plane of the B operand in a stage
    constexpr uint32_t stage_bytes = kPlanes * (kHalf + b_bytes);

    if (warp == 0) nml::tmem_alloc(nml::smem_u32(&tmem_base), 512);
    if (tid == 32) {
        for (int s = 0; s < P.stages; ++s) {
            nml::mbar_init(nml::smem_u32(&full_bar[s]), 1);
            nml::mbar_init(nml::smem_u32(&empty_bar[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            nml::mbar_init(nml::smem_u32(&tfull_bar[b]), 1);
            nml::mbar_init(nml::smem_u32(&tempty_bar[b]), kEpilogueWarps);
        }
        nml::mbar_init(nml::smem_u32(&drain_bar), 1);
        nml::fence_mbar_init();
        nml::abort_state_init(abort_flag, 0);
    }
    pdl_enter();
    const bool skip = skipped(P.c.skip);
    for (int i = tid; i < P.c.count; i += kThreads) {
        const Work* w = P.c.table + i;
        auto word = [](const uint32_t* p) { return static_cast<uint32_t>(load_global(reinterpret_cast<const int*>(p))); };
        first[i] = load_global(kWide ? &w->first_update : &w->first_gram) * (kWide ? 1 : P.jobs);
        info[i] = {load_global(&w->s.m), load_global(&w->s.n), load_global(&w->nb), load_global(&w->wide), {word(&w->x[0]), word(&w->x[1])},
                   word(&w->sym), load_global(&w->sx)};
    }
    nml::tc_fence_before();
    __syncthreads();
    nml::tc_fence_after();
    const uint32_t tmem = tmem_base;
    const int tiles = skip ? 0 : P.tiles;

    auto tile_of = [&](int t) {
        Tile r;
        r.k = owner_of(first, P.c.count, t);
        t -= first[r.k];
        const Info& w = info[r.k];
        r.extra = r.job = 0;
        if (kWide) {
            const int per = (w.nb + w.wide - 1) / w.wide;
            r.i = t / per;
            r.j = t % per * w.wide;
            r.groups = min(2 * w.wide, (w.n - r.j * kBlock + 63) / 64);
            r.slices = (w.m + 63) / 64;
            if (kPlanes == 1) r.extra = min(2, r.slices - 2 * r.i);
        } else {
            const int mb = (w.m + kBlock - 1) / kBlock;
            if (t >= lower(mb, 0)) t -= lower(mb, 0), r.job = 1;
            r.i = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
            while (lower(r.i, 0) > t) --r.i;
            while (lower(r.i + 1, 0) <= t) ++r.i;
            r.j = t - lower(r.i, 0);
            r.groups = 2;
            r.slices = ((P.gram ? w.n : w.m) + 63) / 64;
        }
        return r;
    };
    auto symmetric_first = [&](const Info& w, int buffer) { return w.sym + buffer * lower((w.m + kBlock - 1) / kBlock, 0); };

    if (warp == 0) {
        // ------------------------------------------------------------ producer: a lane to a copy of 8 KB
        int s = 0, issued = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const Tile tile = tile_of(t);
            const Info w = info[tile.k];
            const bool same = P.gram && tile.i == tile.j;
            const int b_pieces = same ? 0 : tile.groups, pieces = kPlanes * (2 + b_pieces);
            // this lane's copy: operand, plane, piece
            const bool is_a = lane < 2 * kPlanes;
            const int at = is_a ? lane : lane - 2 * kPlanes, per = is_a ? 2 : max(1, b_pieces);
            const int plane = at / per, piece = at % per;
            const uint32_t dst = (is_a ? plane * kHalf : kPlanes * kHalf + plane * b_bytes) + piece * kPiece;
            const uint32_t buffer = symmetric_first(w, kWide ? P.left : is_a ? P.job[tile.job].left : P.job[tile.job].right);
            const uint32_t x = w.x[P.from];
            for (int q = 0; q < tile.slices + tile.extra; ++q) {
                if (!__all_sync(0xffffffffu, nml::mbar_wait(nml::smem_u32(&empty_bar[s]), parity ^ 1, abort_flag, P.err, nml::ERR_WAIT_EMPTY))) {
                    ok = false;
                    break;
                }
                const uint32_t bar = nml::smem_u32(&full_bar[s]), to = nml::smem_u32(smem) + s * stage_bytes + dst;
                if (lane == 0) nml::mbar_arrive_expect_tx(bar, pieces * kPiece);
                __syncwarp();
                if (lane < pieces) {
                    const bool low = q >= tile.slices;  // a I times X's low half
                    const int kq = low ? 2 * tile.i + q - tile.slices : q, kb = kq >> 1, h = kq & 1;
                    const uint8_t* from;
                    const uint32_t straight = (h * 2 + piece) * kPiece, across = (piece * 2 + h) * kPiece;  // K-major; MN-major
                    auto symmetric = [&](int row) {
                        return kb <= row ? block_at(P.c.blocks, buffer, lower(row, kb)) + straight : block_at(P.c.blocks, buffer, lower(kb, row)) + across;
                    };
                    if (!kWide) {
                        const int row = is_a ? tile.i : tile.j;
                        from = P.gram ? block_at(P.c.blocks, x, row * w.nb + kb) + straight : symmetric(row);
                    } else if (is_a) {
                        from = low ? block_at(P.c.blocks, P.identity, 0) + straight : symmetric(tile.i);
                    } else {  // X's rows along K: two 64-column groups to a block
                        from = block_at(P.c.blocks, x, kb * w.nb + tile.j + (piece >> 1)) + (low ? kPlane : 0) + ((piece & 1) * 2 + h) * kPiece;
                    }
                    nml::bulk_load(to, from + plane * kPlane, kPiece, bar);
                }
                __syncwarp();
                ++issued;
                if (++s == P.stages) s = 0, parity ^= 1;
            }
        }
        if (!ok || *abort_flag) {  // no copy may be in flight when the block's shared memory goes away
            for (int back = min(issued, P.stages); back > 0; --back) {
                if (--s < 0) s = P.stages - 1, parity ^= 1;
                const uint64_t t0 = nml::globaltimer_ns();
                while (!nml::mbar_try_wait(nml::smem_u32(&full_bar[s]), parity)) {
                    if (nml::globaltimer_ns() - t0 > 2000000ull) {
                        if (lane == 0) atomicCAS(P.err, 0, nml::ERR_WAIT_DRAIN);
                        break;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA
        int s = 0, buf = 0;
        uint32_t parity = 0, tparity = 0;
        bool ok = true;
        const uint32_t ring = nml::smem_u32(smem);
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const Tile tile = tile_of(t);
            const bool same = P.gram && tile.i == tile.j;
            const int slices = tile.slices + tile.extra;
            for (int q = 0; q < slices; ++q) {
                if (kPlanes == 2 || q == 0) {
                    if (!__all_sync(0xffffffffu, nml::mbar_wait(nml::smem_u32(&tempty_bar[buf]), tparity ^ 1, abort_flag, P.err, nml::ERR_WAIT_TMEM_EMPTY))) {
                        ok = false;
                        break;
                    }
                    nml::tc_fence_after();
                }
                if (!__all_sync(0xffffffffu, nml::mbar_wait(nml::smem_u32(&full_bar[s]), parity, abort_flag, P.err, nml::ERR_WAIT_FULL))) {
                    ok = false;
                    break;
                }
                nml::tc_fence_after();
                const bool low = q >= tile.slices, last = kPlanes == 2 || q + 1 == slices;
                const int kb = q >> 1;
                const int a_mn = !P.gram && !low && kb > tile.i;
                const int b_mn = kWide ? 1 : !P.gram && kb > tile.j;
                const uint32_t idesc = nml::make_instr_desc(0, a_mn, b_mn, 128, tile.groups * 64);
                const uint32_t sa = ring + s * stage_bytes, sb = same ? sa : sa + kPlanes * kHalf, bp = same ? kHalf : b_bytes;
                if (nml::elect_one()) {
#pragma unroll
                    for (int p = kPlanes == 2 ? 2 : 0; p >= 0; --p) {  // low x high, high x low, high x high
                        const uint32_t pa = p == 2, pb = p == 1;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint64_t ad = nml::make_smem_desc(sa + pa * kHalf + k * (a_mn ? 2048 : 32), kPiece, 1024, 2);
                            const uint64_t bd = nml::make_smem_desc(sb + pb * bp + k * (b_mn ? 2048 : 32), kPiece, 1024, 2);
                            nml::umma_f16(tmem + buf * 256, ad, bd, idesc, kPlanes == 2 ? k > 0 || p < 2 : k > 0 || q > 0);
                        }
                    }
                    nml::umma_commit(nml::smem_u32(&empty_bar[s]));
                    if (last) nml::umma_commit(nml::smem_u32(&tfull_bar[buf]));
                }
                __syncwarp();
                if (++s == P.stages) s = 0, parity ^= 1;
                if (last && ++buf == 2) buf = 0, tparity ^= 1;
            }
        }
        if (!ok) {  // the products issued so far still read shared memory and write TMEM
            if (nml::elect_one()) nml::umma_commit(nml::smem_u32(&drain_bar));
            __syncwarp();
            const uint64_t t0 = nml::globaltimer_ns();
            while (!nml::mbar_try_wait(nml::smem_u32(&drain_bar), 0)) {
                if (nml::globaltimer_ns() - t0 > 2000000ull) {
                    if (lane == 0) atomicCAS(P.err, 0, nml::ERR_WAIT_DRAIN);
                    break;
                }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue: a thread to a row and half of the columns of the tile
        constexpr int kGroups16 = kWide ? 8 : 4;  // of sixteen columns, to a thread
        int buf = 0;
        uint32_t tparity = 0;
        const int quarter = warp & 3, row = quarter * 32 + lane, side = (warp - 2) >> 2;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
            const Tile tile = tile_of(t);
            const Info w = info[tile.k];
            const int g0 = side * (tile.groups * 2);  // this thread's first sixteen columns; as many for the other side
            const int chunks = kPlanes == 2 ? tile.slices : 1, mine = tile.groups * 2;
            float acc[kGroups16][16];
#pragma unroll
            for (int c = 0; c < kGroups16; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[c][e] = 0.f;
            for (int q = 0; q < chunks; ++q) {
                if (!__all_sync(0xffffffffu, nml::mbar_wait(nml::smem_u32(&tfull_bar[buf]), tparity, abort_flag, P.err, nml::ERR_WAIT_TMEM_FULL))) {
                    ok = false;
                    break;
                }
                nml::tc_fence_after();
                const uint32_t from = tmem + buf * 256 + g0 * 16 + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < kGroups16; ++c) {
                    if (c < mine) {
                        uint32_t r[16];
                        nml::tmem_ld_32x16(from + c * 16, r);
                        nml::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[c][e] += __uint_as_float(r[e]);
                    }
                }
                nml::tc_fence_before();
                __syncwarp();
                if (lane == 0) nml::mbar_arrive(nml::smem_u32(&tempty_bar[buf]));
                if (++buf == 2) buf = 0, tparity ^= 1;
            }
            if (!ok) break;
            const int i = tile.i * kBlock + row;
            if (kKind == RESULT) {
                const Source* src = &P.c.table[tile.k].s;
                const int m = w.m, j0 = tile.j * kBlock + g0 * 16;
                const long long step = load_wide(&src->out_j), at = i * load_wide(&src->out_i) + j0 * step;
                uint8_t* const out = reinterpret_cast<uint8_t*>(load_wide(reinterpret_cast<const long long*>(&src->out)));
                uint8_t* const half = reinterpret_cast<uint8_t*>(load_wide(reinterpret_cast<const long long*>(&src->half)));
                const float f0 = P.f0 / w.sx, rate = P.rate * load_global(&src->scale);  // (a power of two)
                const int in_row = i < m ? min(mine * 16, w.n - j0) : 0;  // this thread's elements
#pragma unroll
                for (int c = 0; c < kGroups16; ++c) {
                    if (c * 16 >= in_row) continue;
                    float v[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) v[q] = acc[c][q] * f0;
                    const long long e = at + c * 16 * step;
                    const int count = in_row - c * 16;
                    if (P.apply) apply16(reinterpret_cast<float*>(out) + e, half ? reinterpret_cast<__half*>(half) + e : nullptr, step, count, v, P.keep, rate);
                    else if (P.out_half) write16(reinterpret_cast<__half*>(out) + e, step, count, v);
                    else write16(reinterpret_cast<float*>(out) + e, step, count, v);
                }
            } else {
                const Symmetric& job = P.job[tile.job];
                const uint32_t to = kKind == ITERATE ? w.x[P.from ^ 1] : symmetric_first(w, job.out), poly = symmetric_first(w, kPoly);
                const int block = kKind == ITERATE ? tile.i * w.nb + tile.j : lower(tile.i, tile.j);
                const float over = P.gram ? 1.f / (w.sx * w.sx) : 1.f;  // (a power of two)
                const float f0 = (kKind == ITERATE ? P.f0 : job.f0) * over, f1 = P.f1 * over;
                const int diagonal = kKind != ITERATE && tile.i == tile.j ? row - g0 * 16 : -1;  // column of the diagonal, among this thread's
#pragma unroll
                for (int c = 0; c < kGroups16; ++c) {
                    if (c >= mine) continue;
                    const int g = g0 + c, half = g >> 2, at16 = (g & 3) * 2;
                    float v[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        v[q] = acc[c][q] * f0;
                        if (kKind == PLAIN && c * 16 + q == diagonal) v[q] += job.d1;
                    }
                    uint8_t* const at = block_at(P.c.blocks, to, block + (half >> 1)) + (half & 1) * kHalf;
                    store16<kKind == ITERATE || kPlanes == 2>(at, row, at16, v);
                    if (kKind == POLY) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            v[q] = acc[c][q] * f1;
                            if (c * 16 + q == diagonal) v[q] += P.d1;
                        }
                        store16<kPlanes == 2>(block_at(P.c.blocks, poly, block) + half * kHalf, row, at16, v);
                    }
                }
            }
        }
    }
    nml::tc_fence_before();
    __syncthreads();
    nml::tc_fence_after();
    if (warp == 0) {
        nml::tmem_relinquish();
        nml::tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- parameters that are no matrices --
constexpr int kVectors = 128;
struct Vector {
    float* param;
    const float* grad;
    float* momentum;
    __half* half;
    int n;
};
struct VectorParams {
    Vector v[kVectors];
    Momentum mo;
    float keep, rate;
    const int* skip;
};
// Plain momentum: p = p keep - rate u, a block to a vector.
__global__ void __launch_bounds__(256) momentum_vectors_kernel(const __grid_constant__ VectorParams P) {
    pdl_enter();
    if (skipped(P.skip)) return;
    const Vector& s = P.v[blockIdx.x];
    for (int e = threadIdx.x; e < s.n; e += 256) {
        const float g = load_global(s.grad + e) * P.mo.inv_scale;
        const float b = P.mo.momentum * load_global(s.momentum + e) + g;
        const float p = load_global(s.param + e) * P.keep - P.rate * (P.mo.nesterov ? g + P.mo.momentum * b : b);
        s.momentum[e] = b;
        s.param[e] = p;
        if (s.half) s.half[e] = __float2half_rn(p);
    }
}

// ---------------------------------------------------------------- host --
static inline size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }

// The steps' coefficients, and powers of two that keep every stored matrix below fp16's largest value.
//
// Chains.  A step's Gram matrix follows from the last one's: with U = U_k of A_k, A_(k+1) = U A_k U (all are polynomials of the first A), and
// X_(k+t) = Q X_k with Q = U_(k+t-1) ... U_k.  So t steps need one product X X^T and one Q X over the long side, and products of
// m x m matrices, half of each, in between: for 5 steps as 3 + 2 and n = r m it is 6 r + 14 instead of 15 r + 5 products of m^3.
// What limits t is that the error of A_k, 2^-24 of its elements, grows by U^2 a step; kGrowth holds the chain's to that of one step from
// a matrix 150 times as large.  (fp32 accuracy, against 64 bits: 3 + 2 as exact as five single steps over gradients of five kinds, 1e-6 to 8e-6;
// all five in one chain 1e-6 to 4e-4.)  "f16" has no such reserve and takes single steps.
constexpr double kGrowth = 150.0;
struct Step {
    double a, b, c;
    int ea, ep, eu, et, eq;  // A, P, U, T and Q are stored times 2^e
    bool starts, ends;       // a chain
};
struct Polynomial {
    Step step[kMaxSteps];
    int steps = 0;
    bool chained = false;
    double largest = 1.0;    // singular value at the chains' starts, hence element of X
};
static int exponent_below(double bound) {  // largest e with bound * 2^e <= 2^15
    return std::max(-24, std::min(24, static_cast<int>(floor(log2(32768.0 / std::max(bound, 1e-6))))));
}
static bool polynomial(const float* coefficients, int steps, int math, Polynomial* p) {
    constexpr int kPoints = 128;        // singular values, at which the matrices' eigenvalues are followed
    constexpr double kBetween = 1.01;   // and what lies between two of them
    double l = kBetween, lambda[kPoints + 1], q[kPoints + 1], growth = 1.0;
    p->steps = steps;
    p->largest = l;
    bool starts = true;
    for (int k = 0; k < steps; ++k) {
        Step& s = p->step[k];
        s.a = coefficients[3 * k];
        s.b = coefficients[3 * k + 1];
        s.c = coefficients[3 * k + 2];
        if (!(fabs(s.a) < 1e3 && fabs(s.b) < 1e3 && fabs(s.c) < 1e3)) return false;
        if (starts) {
            for (int i = 0; i <= kPoints; ++i) lambda[i] = l * i / kPoints * (l * i / kPoints), q[i] = 1.0;
            growth = 1.0;
        }
        double ma = 0, mp = 0, mu = 0, mt = 0, mq = 0, next = 0;
        for (int i = 0; i <= kPoints; ++i) {
            const double u = s.a + lambda[i] * (s.b + s.c * lambda[i]);
            ma = std::max(ma, lambda[i]);
            mp = std::max(mp, fabs(s.b + s.c * lambda[i]));
            mu = std::max(mu, fabs(u));
            mt = std::max(mt, fabs(u * lambda[i]));
            q[i] *= u;
            mq = std::max(mq, fabs(q[i]));
            lambda[i] *= u * u;
            next = std::max(next, lambda[i]);
        }
        s.starts = starts;
        s.ea = exponent_below(ma * kBetween * kBetween);
        s.ep = exponent_below(mp * kBetween);
        s.eu = exponent_below(mu * kBetween);
        s.et = exponent_below(mt * kBetween * kBetween);
        s.eq = exponent_below(mq * kBetween);
        growth *= std::max(1.0, mu * mu);
        if (!(next <= 4096.0)) return false;  // singular values beyond 64
        s.ends = math == NML_MATH_F16 || k == steps - 1 || growth > kGrowth;
        starts = s.ends;
        if (!s.ends) p->chained = true;
        if (s.ends) l = std::max(sqrt(next) * kBetween, 1e-3), p->largest = std::max(p->largest, l);
    }
    return true;
}

struct Plan {
    int sums = 0, halves = 0, gram_tiles = 0, update_tiles = 0;
    uint32_t blocks = 0, identity = 0;
    size_t table_at = 0, sums_at = 0, blocks_at = 0, bytes = 0;
};
// Lays a group of at most kGroup matrices out; the sources' sizes are set.
static Plan plan_group(Work* w, int count, int math, const Polynomial& poly, int sms) {
    Plan p;
    long long wide_tiles = 0;
    for (int k = 0; k < count; ++k) {
        w[k].mb = (w[k].s.m + kBlock - 1) / kBlock;
        w[k].nb = (w[k].s.n + kBlock - 1) / kBlock;
        wide_tiles += static_cast<long long>(w[k].mb) * ((w[k].nb + 1) / 2);
    }
    for (int k = 0; k < count; ++k) {
        Work& v = w[k];
        const long long elements = static_cast<long long>(v.s.m) * v.s.n;
        v.first_sum = p.sums;
        v.sums = static_cast<int>((elements + kSumElements - 1) / kSumElements);
        p.sums += v.sums;
        v.first_half = p.halves;
        p.halves += v.mb * v.nb * 2;
        v.first_gram = p.gram_tiles;
        p.gram_tiles += v.mb * (v.mb + 1) / 2;
        v.wide = wide_tiles >= sms ? 2 : 1;
        v.first_update = p.update_tiles;
        p.update_tiles += v.mb * ((v.nb + v.wide - 1) / v.wide);
        for (uint32_t* at : {&v.x[0], &v.x[1]}) *at = p.blocks, p.blocks += v.mb * v.nb;
        v.sym = p.blocks;
        p.blocks += (poly.chained ? 7 : 3) * (v.mb * (v.mb + 1) / 2);
        const int e = std::min(exponent_below(poly.largest), static_cast<int>(lround(0.5 * log2(static_cast<double>(elements)))));
        v.sx = static_cast<float>(ldexp(1.0, e));
    }
    p.identity = p.blocks;
    if (math == NML_MATH_F16) p.blocks += poly.steps;
    p.sums_at = round_up(sizeof(Work) * kGroup, 256);
    p.blocks_at = p.sums_at + round_up(sizeof(double) * p.sums, 1024);
    p.bytes = p.blocks_at + static_cast<size_t>(p.blocks) * 2 * kPlane;
    return p;
}

typedef void (*ProductKernel)(const ProductParams);
static ProductKernel product_kernel(int planes, int kind) {
    if (planes == 1)
        return kind == POLY ? ortho_product_kernel<1, POLY> : kind == PLAIN ? ortho_product_kernel<1, PLAIN>
               : kind == ITERATE ? ortho_product_kernel<1, ITERATE> : ortho_product_kernel<1, RESULT>;
    return kind == POLY ? ortho_product_kernel<2, POLY> : kind == PLAIN ? ortho_product_kernel<2, PLAIN>
           : kind == ITERATE ? ortho_product_kernel<2, ITERATE> : ortho_product_kernel<2, RESULT>;
}

struct Call {
    int in_dtype = NML_F32, out_dtype = NML_F32, math = NML_MATH_3XF16;
    float eps = 0.f;
    Momentum mo = {1.f, 0.f, false, false};
    bool apply = false;
    float keep = 0.f, rate = 0.f;
    const int* skip = nullptr;
};

template <int N>
static void launch_sums(const Work* w, int count, const Call& call, const Plan& p, Work* table, double* sums, cudaStream_t st) {
    Group<N> g;
    std::copy(w, w + count, g.w);
    if (call.in_dtype == NML_F16)
        nml::launch(ortho_sums_kernel<N, __half>, p.sums, 256, 0, st, g, count, call.mo, table, sums, call.skip);
    else
        nml::launch(ortho_sums_kernel<N, float>, p.sums, 256, 0, st, g, count, call.mo, table, sums, call.skip);
}

// One group: the launches of all its steps.
static int run_group(Work* w, int count, const Call& call, const Polynomial& poly, void* workspace, size_t bytes, cudaStream_t st) {
    int* err;
    int sms;
    if (const int rc = nml::current_device(&err, &sms)) return rc;
    const Plan p = plan_group(w, count, call.math, poly, sms);
    uint8_t* const base = reinterpret_cast<uint8_t*>(round_up(reinterpret_cast<uintptr_t>(workspace), 1024));
    if (!workspace || base + p.bytes > static_cast<uint8_t*>(workspace) + bytes) return NML_ERR_WORKSPACE;
    Work* const table = reinterpret_cast<Work*>(base);
    double* const sums = reinterpret_cast<double*>(base + p.sums_at);
    if (count <= 8) launch_sums<8>(w, count, call, p, table, sums, st);
    else launch_sums<kGroup>(w, count, call, p, table, sums, st);
    const Common common = {table, sums, base + p.blocks_at, call.skip, count};
    PackParams pack = {common, call.mo, call.eps, p.halves, p.identity, {}};
    for (int k = 0; k < poly.steps; ++k) pack.diagonal[k] = static_cast<float>(ldexp(poly.step[k].a, poly.step[k].eu));
    const int pack_grid = p.halves + (call.math == NML_MATH_F16 ? 2 * poly.steps : 0);
    nml::launch(call.in_dtype == NML_F16 ? ortho_pack_kernel<__half> : ortho_pack_kernel<float>, pack_grid, 256, 0, st, pack);
    const int planes = call.math == NML_MATH_F16 ? 1 : 2;
    int launched = 2, from = 0;
    auto product = [&](int kind, ProductParams& q) {
        const bool wide = kind >= ITERATE;
        q.c = common;
        q.err = err;
        q.jobs = std::max(q.jobs, 1);
        q.tiles = wide ? p.update_tiles : p.gram_tiles * q.jobs;
        q.stages = std::min<int>(kMaxStages, kStageBytes / (planes * (wide ? 3 * kHalf : 2 * kHalf)));
        q.from = from;
        nml::launch(product_kernel(planes, kind), std::min(q.tiles, sms), kThreads, kProductSmem, st, q);
        ++launched;
    };
    // a product of two symmetric matrices stored times 2^el and 2^er, to be stored times 2^eo, + d on the diagonal
    auto symmetric = [](int left, int el, int right, int er, int out, int eo, double d) {
        return Symmetric{left, right, out, static_cast<float>(ldexp(1.0, eo - el - er)), static_cast<float>(ldexp(d, eo))};
    };
    int u = kUpdate, q_at = kQ;       // the current U and Q
    int eq = 0, eu_last = 0;          // Q's exponent; that of the last step's U, which is in the other buffer
    for (int k = 0; k < poly.steps; ++k) {
        const Step& s = poly.step[k];
        {   // A and P
            ProductParams q = {};
            q.gram = s.starts;
            if (s.starts) q.job[0].out = kGram, q.job[0].f0 = static_cast<float>(ldexp(1.0, s.ea));
            else q.job[0] = symmetric(u, eu_last, kT, poly.step[k - 1].et, kGram, s.ea, 0.0);
            const double f = s.starts ? 1.0 : ldexp(1.0, -eu_last - poly.step[k - 1].et);
            q.f1 = static_cast<float>(ldexp(s.c * f, s.ep));
            q.d1 = static_cast<float>(ldexp(s.b, s.ep));
            product(POLY, q);
        }
        {   // U
            if (!s.starts) u = u == kUpdate ? kUpdate2 : kUpdate;
            if (s.starts) q_at = u, eq = s.eu;
            ProductParams q = {};
            q.job[0] = symmetric(kPoly, s.ep, kGram, s.ea, u, s.eu, s.a);
            product(PLAIN, q);
            eu_last = s.eu;
        }
        {   // Q = U Q, and T = U A where the chain goes on
            ProductParams q = {};
            if (!s.ends) q.job[q.jobs++] = symmetric(u, s.eu, kGram, s.ea, kT, s.et, 0.0);
            if (!s.starts) {
                const int to = q_at == kQ ? kQ2 : kQ;
                q.job[q.jobs++] = symmetric(u, s.eu, q_at, eq, to, s.eq, 0.0);
                q_at = to;
                eq = s.eq;
            }
            if (q.jobs) product(PLAIN, q);
        }
        if (s.ends) {
            const bool last = k == poly.steps - 1;
            ProductParams q = {};
            q.left = q_at;
            q.f0 = static_cast<float>(ldexp(1.0, -eq));
            q.identity = p.identity + k;
            q.out_half = call.out_dtype == NML_F16;
            q.apply = call.apply;
            q.keep = call.keep;
            q.rate = call.rate;
            product(last ? RESULT : ITERATE, q);
            from ^= 1;
        }
    }
    NMLO_CUDA(cudaGetLastError());
    nml::count_launches(launched);
    return NML_OK;
}

static bool math_ok(int math) { return math == NML_MATH_F16 || math == NML_MATH_3XF16; }
static bool size_ok(int rows, int cols) {
    // (indexes of blocks, tiles and sums are 32-bit)
    return rows > 0 && cols > 0 && static_cast<long long>(rows) * cols <= (1ll << 36);
}
static void set_sizes(Source& s, int rows, int cols) {
    s.m = std::min(rows, cols);
    s.n = std::max(rows, cols);
}
static bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Whether what a step writes is in one place each: a parameter that is listed twice would be updated by two blocks at a time.
static bool apart(const nml_muon_param* params, int count) {
    typedef std::pair<uintptr_t, uintptr_t> Range;
    try {
        std::vector<Range> r;
        r.reserve(3 * static_cast<size_t>(count));
        for (int k = 0; k < count; ++k) {
            const uintptr_t n = static_cast<uintptr_t>(std::max(params[k].rows, 1)) * params[k].cols;
            auto add = [&](const void* p, size_t size) {
                if (p) r.emplace_back(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + n * size);
            };
            add(params[k].param, 4);
            add(params[k].momentum, 4);
            add(params[k].param_f16, 2);
        }
        std::sort(r.begin(), r.end());
        for (size_t k = 1; k < r.size(); ++k)
            if (r[k].first < r[k - 1].second) return false;
        return true;
    } catch (...) {
        return false;
    }
}

// Workspace of the largest group of `count` matrices whose sizes `size(k, source)` sets (false: not a matrix, left out).
template <class F>
static int workspace_of(int count, int math, int steps, F&& size, size_t* bytes) {
    Polynomial poly;
    poly.steps = steps;
    poly.chained = math != NML_MATH_F16 && steps > 1;  // (whether they are depends on the coefficients)
    Work w[kGroup];
    *bytes = 0;
    int sms = nml::usable_sms(), filled = 0;
    for (int k = 0; k <= count; ++k) {
        if (filled == kGroup || (k == count && filled > 0)) {
            *bytes = std::max(*bytes, plan_group(w, filled, math, poly, sms).bytes + 1024);
            filled = 0;
        }
        if (k < count) {
            w[filled] = Work();
            if (size(k, w[filled].s)) ++filled;
        }
    }
    return NML_OK;
}

}  // namespace nml_ortho

using namespace nml_ortho;

int nml::prepare_ortho_kernels() {
    for (int planes = 1; planes <= 2; ++planes)
        for (int kind = POLY; kind <= RESULT; ++kind)
            NMLO_CUDA(cudaFuncSetAttribute(product_kernel(planes, kind), cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kProductSmem)));
    cudaFuncAttributes a;
    const void* others[] = {(const void*)ortho_sums_kernel<8, float>, (const void*)ortho_sums_kernel<8, __half>,
                            (const void*)ortho_sums_kernel<kGroup, float>, (const void*)ortho_sums_kernel<kGroup, __half>,
                            (const void*)ortho_pack_kernel<float>, (const void*)ortho_pack_kernel<__half>, (const void*)momentum_vectors_kernel};
    for (const void* f : others) NMLO_CUDA(cudaFuncGetAttributes(&a, f));
    return NML_OK;
}

extern "C" {

int nml_orthogonalize_workspace_size(const nml_matrix* matrices, int count, int math, int steps, size_t* bytes) {
    if (!bytes || count < 0 || (count > 0 && !matrices) || !math_ok(math) || steps < 1 || steps > kMaxSteps) return NML_ERR_INVALID;
    for (int k = 0; k < count; ++k)
        if (!size_ok(matrices[k].rows, matrices[k].cols)) return NML_ERR_INVALID;
    return workspace_of(count, math, steps, [&](int k, Source& s) { return set_sizes(s, matrices[k].rows, matrices[k].cols), true; }, bytes);
}

int nml_orthogonalize(const nml_matrix* matrices, int count, int in_dtype, int out_dtype, int math, int steps, const float* coefficients,
                      float eps, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    if (const int rc = nml_orthogonalize_workspace_size(matrices, count, math, steps, &need)) return rc;
    if ((in_dtype != NML_F32 && in_dtype != NML_F16) || (out_dtype != NML_F32 && out_dtype != NML_F16) || !coefficients || !(eps >= 0.f)) return NML_ERR_INVALID;
    for (int k = 0; k < count; ++k) {
        const nml_matrix& x = matrices[k];
        if (!x.in || !x.out || !aligned_to(x.in, in_dtype == NML_F16 ? 2 : 4) || !aligned_to(x.out, out_dtype == NML_F16 ? 2 : 4)) return NML_ERR_INVALID;
        auto dense = [&](long long r, long long c) {  // one of the two runs through memory, the other by steps that do not overlap
            return (c == 1 && r >= x.cols) || (r == 1 && c >= x.rows) || (x.rows == 1 && c == 1) || (x.cols == 1 && r == 1);
        };
        if (!dense(x.in_row, x.in_col) || !dense(x.out_row, x.out_col)) return NML_ERR_INVALID;
    }
    Polynomial poly;
    if (!polynomial(coefficients, steps, math, &poly)) return NML_ERR_UNSUPPORTED;
    if (count > 0 && (!workspace || workspace_bytes < need)) return NML_ERR_WORKSPACE;
    Call call;
    call.in_dtype = in_dtype;
    call.out_dtype = out_dtype;
    call.math = math;
    call.eps = eps;
    Work w[kGroup];
    for (int at = 0; at < count; at += kGroup) {
        const int n = std::min(kGroup, count - at);
        for (int k = 0; k < n; ++k) {
            const nml_matrix& x = matrices[at + k];
            const bool turn = x.rows > x.cols;
            w[k] = Work();
            w[k].s = {x.in, x.out, nullptr, nullptr, turn ? x.in_col : x.in_row, turn ? x.in_row : x.in_col,
                      turn ? x.out_col : x.out_row, turn ? x.out_row : x.out_col, 0, 0, 1.f};
            set_sizes(w[k].s, x.rows, x.cols);
        }
        if (const int rc = run_group(w, n, call, poly, workspace, workspace_bytes, static_cast<cudaStream_t>(stream))) return rc;
    }
    return NML_OK;
}

int nml_muon_workspace_size(const nml_muon_param* params, int count, int math, int steps, size_t* bytes) {
    if (!bytes || count < 0 || (count > 0 && !params) || !math_ok(math) || steps < 1 || steps > kMaxSteps) return NML_ERR_INVALID;
    for (int k = 0; k < count; ++k)
        if (params[k].rows < 0 || params[k].cols <= 0 || (params[k].rows > 0 && !size_ok(params[k].rows, params[k].cols))) return NML_ERR_INVALID;
    return workspace_of(count, math, steps, [&](int k, Source& s) { return params[k].rows > 0 && (set_sizes(s, params[k].rows, params[k].cols), true); }, bytes);
}

int nml_muon_step(const nml_muon_param* params, int count, int math, int steps, const float* coefficients, float eps, float lr, float momentum,
                  int nesterov, float weight_decay, float inv_scale, const int* found_inf, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    if (const int rc = nml_muon_workspace_size(params, count, math, steps, &need)) return rc;
    if (!apart(params, count)) return NML_ERR_INVALID;
    if (!coefficients || !(eps >= 0.f) || !aligned_to(found_inf, 4)) return NML_ERR_INVALID;
    for (int k = 0; k < count; ++k) {
        const nml_muon_param& p = params[k];
        if (!p.param || !p.grad || !p.momentum || !aligned_to(p.param, 4) || !aligned_to(p.grad, 4) || !aligned_to(p.momentum, 4) || !aligned_to(p.param_f16, 2))
            return NML_ERR_INVALID;
    }
    Polynomial poly;
    if (!polynomial(coefficients, steps, math, &poly)) return NML_ERR_UNSUPPORTED;
    if (need > 0 && (!workspace || workspace_bytes < need)) return NML_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Call call;
    call.math = math;
    call.eps = eps;
    call.mo = {inv_scale, momentum, true, nesterov != 0};
    call.apply = true;
    call.keep = 1.f - lr * weight_decay;
    call.rate = lr;
    call.skip = found_inf;
    VectorParams vectors = {};
    vectors.mo = call.mo;
    vectors.keep = call.keep;
    vectors.rate = lr;
    vectors.skip = found_inf;
    Work w[kGroup];
    int matrices = 0, others = 0;
    for (int k = 0; k <= count; ++k) {
        if (matrices == kGroup || (k == count && matrices > 0)) {
            if (const int rc = run_group(w, matrices, call, poly, workspace, workspace_bytes, st)) return rc;
            matrices = 0;
        }
        if (others == kVectors || (k == count && others > 0)) {
            int* err;
            int sms;
            if (const int rc = nml::current_device(&err, &sms)) return rc;
            nml::launch(momentum_vectors_kernel, others, 256, 0, st, vectors);
            NMLO_CUDA(cudaGetLastError());
            nml::count_launches(1);
            others = 0;
        }
        if (k == count) break;
        const nml_muon_param& p = params[k];
        if (p.rows == 0) {
            vectors.v[others++] = {p.param, p.grad, p.momentum, static_cast<__half*>(p.param_f16), p.cols};
            continue;
        }
        const long long row = p.cols, col = 1;
        const bool turn = p.rows > p.cols;
        w[matrices] = Work();
        w[matrices].s = {p.grad, p.param, p.momentum, static_cast<__half*>(p.param_f16), turn ? col : row, turn ? row : col,
                         turn ? col : row, turn ? row : col, 0, 0, p.scale};
        set_sizes(w[matrices].s, p.rows, p.cols);
        ++matrices;
    }
    return NML_OK;
}

}  // extern "C"
