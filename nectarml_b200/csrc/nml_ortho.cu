// Orthogonalised updates: a few steps of the iteration
//
//   X <- (a I + b A + c A^2) X,  A = X X^T,  starting at G / (|G| + eps)  (Frobenius norm),
//
// which drive the singular values of G towards 1 and keep its singular vectors, and the optimizer step that applies such an update
// to every matrix of a model (momentum, orthogonalisation, weight decay, fp16 copy).  The reference's optimizers
// (nectarml/optim/sgd.py:60-90) have no such update; this stands beside nml_sgd_momentum_step.
//
// A group of matrices is worked on at once, each turned so that it is wide: X is m x n with m <= n.  A step is three products:
//   A = X X^T         symmetric, the blocks on and below the diagonal, with P = b I + c A beside it
//   U = a I + P A     symmetric too (polynomials of A commute)
//   X = U X           (the last one writes the result, or the parameters, in the caller's layout)
// or, chained, two products X X^T and Q X for several steps (see Polynomial).
//
// One launch runs all products of all matrices: 15 to 17 launches in a row cost a small matrix 8 us each and a group its idle SMs at the
// end of each.  Blocks take tiles from one counter, in an order in which every tile follows those it needs, and wait for
// a matrix's earlier products by a counter of its own; so whatever number of blocks is running, the first waiting tile's predecessors are done or
// being worked on.
//
// Operands are fp16.  |X| <= 1 bounds every element of every matrix here, so powers of two chosen on the host put all of them
// into fp16's range; of the data only |G| next to eps matters to that (see lift_of).
//   "3xf16" (fp32 results): every operand is a high and a low half, 22 bits, and a product is the three that matter, in fp32
//           accumulators: an error of about 2^-22 of the largest element a product.  Five single steps are 1.0e-6 to 2.4e-6 off, fp32's 1.0e-6 to
//           3.5e-6 (65 x 65 to 1600 x 1700); chained ones (see Polynomial) a third to four times as much as fp32's.
//   "f16"   one product.  What may not be rounded to 11 bits is X itself where it is carried from step to step: noise in directions whose singular
//           value is small grows by `a` a step (3.4^5 = 490), the signal in the others does not.  So X keeps its low half, and the
//           update adds a I times it: one more K block a tile.  (Errors of the result against 64 bits at gradients of 32 strong
//           directions, 512 x 512: 1.0e-3; with X rounded 5.9e-3; all of U X in two products 1.2e-3.)
//
// Storage.  Every matrix between the products lies in blocks of 128 x 128, a block as two halves of 64 columns, each 128
// rows of 128 bytes in the 128-byte swizzle that tcgen05.mma reads: a tile of an operand is contiguous, an untiled bulk copy brings it (a
// tiled one where two blocks work together and the copy signals the other one's barrier) and ragged sizes are zeros in the blocks.  Such a half serves as K-major (its rows are the M or
// N index) and as MN-major operand (its columns are), so X is read both ways, and a block of a symmetric matrix
// stands for its mirror image too.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <iterator>
#include <type_traits>
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

constexpr int kGroup = 64;             // matrices of one run of launches
constexpr int kMaxSteps = 32;
constexpr int kBlock = 128;            // rows and columns of a block
constexpr uint32_t kHalf = 16384;      // bytes of one half of a block
constexpr uint32_t kPiece = 8192;      // of one copy: 64 rows of a half
constexpr uint32_t kPlane = 2 * kHalf; // of a block
constexpr int kSumElements = 8192;     // of a block of the sum of squares

// Symmetric matrices of a step, as buffers of the workspace: A, P, and U where every step has its own; T = U A, a second U and two Q (see
// Polynomial) where steps are chained.
enum { kGram = 0, kPoly = 1, kUpdate = 2, kUpdate2 = 3, kT = 4, kQ = 5, kQ2 = 6 };

// What a product's epilogue makes of the accumulators D.
enum {
    POLY = 0,    // symmetric: A = D f0, and P = D f1 + d1 I beside it
    PLAIN = 1,   // symmetric: D f0 + d1 I
    ITERATE = 2, // X = D f1
    RESULT = 3,  // D f1 in the caller's layout, or the parameters' update
    SUM = 4      // POLY of a matrix's partial products X X^T, which POLY left in fp32 where K is in several parts
};
struct Symmetric {  // buffers of one symmetric product
    int left, right, out;
    float f0, d1;
};
// A product of every matrix of a class.
struct Op {
    int kind, jobs;            // of symmetric products: the tiles of a second one follow those of the first
    int gram, from;            // POLY: of X X^T; which copy of X is read
    int grown;                 // log2 of what the steps may have multiplied that X by, and in higher bits, of what they may have the one that is written
    Symmetric job[2];
    float f1, d1;
    int left;                  // ITERATE, RESULT: the symmetric factor
    uint32_t identity;         // "f16": block of this step's a I
    int gram_before, symmetric_before, wide_before, sum_before;  // what of the class is in front of this one
};
// Matrices whose steps are chained and those whose steps are single run different products; a round is one product of each.
constexpr int kClasses = 2;
constexpr int kMaxRounds = 5 * kMaxSteps;
struct Round {
    int first, of_first;       // tiles of all rounds in front, of the first class in this one
    Op op[kClasses];
};

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
    uint32_t x[2], sym, partial;        // first blocks of X's two copies, the symmetric matrices and partial products, in blocks of two planes
    int mb, nb;                         // blocks along m and n
    int first_sum, sums;                // its partial sums of squares
    int first_half;                     // its halves of X
    int first_gram, first_symmetric, first_update, first_parts;  // its tiles: of X X^T, symmetric products, Q X, SUM
    int wide;                           // 64-column groups to a tile of Q X: 1, 2 or 4
    int fine, parts;                    // tiles to a block of a symmetric product, 1 or 2; parts of K of X X^T
    int sx;                             // X is stored times 2^sx, and more where it is small (see lift)
    int chained;
    int lift;                           // written by the pass that finds the norm (see lift_of), for those behind it
};
template <int N>
struct Group {
    Work w[N];
};

struct Common {
    Work* table;
    double* sums;
    Round* rounds;
    int* done;        // the tile counter, and behind it every matrix's finished eighths of tiles
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

// Where |G| is far below eps, X starts at a norm far below 1, and the halves of its elements would be too few bits of fp16's range (64 bits off by 2e-2 at
// |G| = 1e-6 eps, where fp32 is by 1e-7).  So it is stored times 2^lift more, lift = floor(log2 (|G| + eps) / |G|), less what the steps so far may have
// multiplied it by, as long as that is positive.
constexpr int kMostLift = 100;
__device__ __forceinline__ int lift_of(double own, double norm) {
    if (!(norm >= 2.0 * own) || own == 0.0) return 0;
    const double over = norm / own;
    return over > 1.0 ? min(kMostLift, ilogb(over)) : 0;  // (infinities: none)
}
__device__ __forceinline__ int lifted(int lift, int grown) { return max(0, lift - grown); }
constexpr int kGrownBits = 8;
// 2^e, 0 below fp32's normal range.
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.f : __int_as_float((e + 127) << 23); }

template <typename T>
__device__ __forceinline__ float load_as_float(const T* p) { return static_cast<float>(load_global(p)); }
template <>
__device__ __forceinline__ float load_as_float<__half>(const __half* p) { return __half2float(load_global(p)); }

// ---------------------------------------------------------------- sum of squares --
// Partial sums of squares in double, kSumElements elements a block, in memory order; the optimizer step's momentum on the way.
// The first block leaves the group's table in the workspace and clears the counters.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&v)[4]) {
    const float4 t = load_global(reinterpret_cast<const float4*>(p));
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
}
template <>
__device__ __forceinline__ void load4<__half>(const __half* p, float (&v)[4]) {
    const uint2 t = load_global(reinterpret_cast<const uint2*>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
template <typename T>
__device__ __forceinline__ bool vectors_of_4(const T* p) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; }

__device__ __forceinline__ float moved(const Momentum& mo, float grad, float old, float& next) {
    const float g = grad * mo.inv_scale;
    next = mo.momentum * old + g;
    return mo.nesterov ? g + mo.momentum * next : next;
}

template <int N, typename T>
__global__ void __launch_bounds__(256) ortho_sums_kernel(const __grid_constant__ Group<N> group, const Common c, const Momentum mo) {
    pdl_enter();
    __shared__ double part[8];
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < c.count; i += blockDim.x) c.table[i] = group.w[i];
        for (int i = threadIdx.x; i <= kGroup; i += blockDim.x) c.done[i] = 0;
    }
    if (skipped(c.skip)) return;
    int k = 0;
    {
        int lo = 0, hi = c.count - 1;
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
    const int count = static_cast<int>(min(total - first, static_cast<long long>(kSumElements)));
    const T* in = static_cast<const T*>(s.in);
    double sum = 0.0;
    const bool dense = pitch == inner || total == inner;
    if (dense && count == kSumElements && vectors_of_4(in) && (!mo.on || vectors_of_4(s.momentum))) {
        constexpr int kLoads = kSumElements / 1024;
        float v[kLoads][4];
#pragma unroll
        for (int l = 0; l < kLoads; ++l) load4(in + first + l * 1024 + threadIdx.x * 4, v[l]);
        if (mo.on) {
            float b[kLoads][4];
#pragma unroll
            for (int l = 0; l < kLoads; ++l) load4<float>(s.momentum + first + l * 1024 + threadIdx.x * 4, b[l]);
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[l][q] = moved(mo, v[l][q], b[l][q], b[l][q]);
                reinterpret_cast<float4*>(s.momentum + first + l * 1024)[threadIdx.x] = make_float4(b[l][0], b[l][1], b[l][2], b[l][3]);
            }
        }
#pragma unroll
        for (int l = 0; l < kLoads; ++l)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum += static_cast<double>(v[l][q]) * static_cast<double>(v[l][q]);
    } else {
        const long long outer0 = first / inner;
        const unsigned rest = static_cast<unsigned>(first - outer0 * inner);
#pragma unroll 4
        for (int e = threadIdx.x; e < count; e += 256) {
            const unsigned outer = (rest + e) / inner;
            float v = load_as_float(in + (outer0 + outer) * pitch + (rest + e - outer * inner));
            if (mo.on) v = moved(mo, v, load_global(s.momentum + first + e), s.momentum[first + e]);  // (dense, as the parameter)
            sum += static_cast<double>(v) * static_cast<double>(v);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += part[w];
        c.sums[blockIdx.x] = sum;
    }
}

// ---------------------------------------------------------------- blocks --
__device__ __forceinline__ uint8_t* block_at(uint8_t* blocks, uint32_t first, int index) {
    return blocks + (static_cast<size_t>(first) + index) * (2 * kPlane);
}
// A block on or below the diagonal of a symmetric matrix.
__device__ __forceinline__ int lower(int i, int j) { return i * (i + 1) / 2 + j; }

// High and low halves of eight values.
__device__ __forceinline__ void split8(const float* v, uint4& high, uint4& low) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const __half2 a = __floats2half2_rn(v[2 * q], v[2 * q + 1]);
        const float2 f = __half22float2(a);
        const __half2 b = __floats2half2_rn(v[2 * q] - f.x, v[2 * q + 1] - f.y);
        h[q] = *reinterpret_cast<const uint32_t*>(&a);
        l[q] = *reinterpret_cast<const uint32_t*>(&b);
    }
    high = make_uint4(h[0], h[1], h[2], h[3]);
    low = make_uint4(l[0], l[1], l[2], l[3]);
}
// Place of chunk c of a row in a half of a block: the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }

// ---------------------------------------------------------------- first iterate --
// One half (128 x 64) of X to a block: the matrix over its norm, in two planes, zeros beyond its edges.  The blocks behind write the
// identity blocks of "f16", a_k I for every step, and the last one the rounds.
template <int N>
struct PackParams {
    Common c;
    Momentum mo;
    float eps;
    int halves, rounds;
    uint32_t identity;  // first block
    int identities;
    float diagonal[kMaxSteps];
    Round round[N];
};
// (five blocks an SM: 48 registers, hence more loads in flight than the 40 that fit six.  MLP step's 34 million elements 84 -> 75 us)
template <int N, typename T>
__global__ void __launch_bounds__(256, 5) ortho_pack_kernel(const __grid_constant__ PackParams<N> P) {
    pdl_enter();
    if (skipped(P.c.skip)) return;
    __shared__ float tile[64][129];
    __shared__ double part[8];
    __shared__ int first[kGroup];
    const int tid = threadIdx.x;
    if (static_cast<int>(blockIdx.x) >= P.halves) {
        const int k = blockIdx.x - P.halves, half = k & 1;
        if (k < 2 * P.identities) {
            uint8_t* const out = block_at(P.c.blocks, P.identity, k / 2) + half * kHalf;
            for (int o = tid; o < 128 * 8; o += 256) {
                float v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = half * 64 + (o & 7) * 8 + q == o / 8 ? P.diagonal[k / 2] : 0.f;
                uint4 h, l;
                split8(v, h, l);
                *reinterpret_cast<uint4*>(out + swizzled(o / 8, o & 7)) = h;
            }
        } else {
            for (int o = tid; o < P.rounds; o += 256) P.c.rounds[o] = P.round[o];
        }
        return;
    }
    for (int i = tid; i < P.c.count; i += 256) first[i] = load_global(&P.c.table[i].first_half);
    __syncthreads();
    // (from the last one to the first: the sums have read the matrices in the other order, so the last ones are in L2)
    const int at_half = P.halves - 1 - blockIdx.x, k = owner_of(first, P.c.count, at_half);
    const Work w = load_work(P.c.table + k);
    const Source& s = w.s;
    const int half = at_half - first[k], i0 = half / (2 * w.nb) * kBlock, j0 = half % (2 * w.nb) * 64;
    uint8_t* const out = block_at(P.c.blocks, w.x[0], half / 2) + (half & 1) * kHalf;
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
    const double own = sqrt(sum), norm = own + static_cast<double>(P.eps);
    const int lift = lift_of(own, norm);
    const double inv = norm == 0.0 ? 0.0 : __hiloint2double((1023 + w.sx + lift) << 20, 0) / norm;  // (zeros stay zeros without an eps too)
    if (half == 0 && tid == 0) P.c.table[k].lift = lift;  // (no block of this pass uses what it reads there)
    const T* const in = static_cast<const T*>(s.in);
    auto update = [&](float v, float momentum) {  // of the element's gradient and new momentum
        if (P.mo.on) {
            v *= P.mo.inv_scale;
            v = P.mo.nesterov ? v + P.mo.momentum * momentum : momentum;
        }
        return static_cast<float>(static_cast<double>(v) * inv);
    };
    const bool turned = s.in_i == 1 && s.in_j != 1;
    const long long pitch = turned ? s.in_j : s.in_i;
    const bool vectors = pitch % 4 == 0 && vectors_of_4(in) && (!P.mo.on || vectors_of_4(s.momentum));
    // four elements that lie behind one another in memory, of which `count` exist
    auto four = [&](long long at, int count, float (&v)[4]) {
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (vectors && count >= 4) {
            load4(in + at, v);
            if (P.mo.on) load4<float>(s.momentum + at, b);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q] = q < count ? load_as_float(in + at + q) : 0.f;
                if (P.mo.on && q < count) b[q] = load_global(s.momentum + at + q);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = update(v[q], b[q]);
    };
    if (turned) {
#pragma unroll 2
        for (int j = tid / 32; j < 64; j += 8) {
            const int i = (tid & 31) * 4;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (j0 + j < s.n && i0 + i < s.m) four(i0 + i + (j0 + j) * pitch, s.m - i0 - i, v);
#pragma unroll
            for (int q = 0; q < 4; ++q) tile[j][i + q] = v[q];
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = tid; o < 128 * 8; o += 256) {
        const int row = o >> 3, chunk = o & 7;
        float v[8];
        if (turned) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = tile[chunk * 8 + q][row];
        } else {
            const int i = i0 + row, j = j0 + chunk * 8;
            float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
            if (i < s.m && j < s.n) four(i * pitch + j, s.n - j, a);
            if (i < s.m && j + 4 < s.n) four(i * pitch + j + 4, s.n - j - 4, b);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = a[q], v[4 + q] = b[q];
        }
        uint4 h, l;
        split8(v, h, l);
        *reinterpret_cast<uint4*>(out + swizzled(row, chunk)) = h;
        *reinterpret_cast<uint4*>(out + kPlane + swizzled(row, chunk)) = l;
    }
}

// ---------------------------------------------------------------- products --
// What another block of the same grid has written: past the SM's own cache.
__device__ __forceinline__ float4 load_shared_by_blocks(const float4* p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(__cvta_generic_to_global(p)) : "memory");
    return v;
}
__device__ __forceinline__ long long load_wide(const long long* p) {
    long long v;
    asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(__cvta_generic_to_global(p)));
    return v;
}
// Pairs: the blocks as [plane][half][rows 0 to 63, 64 to 127][16][256 elements], so that one copy brings an operand's slice in both planes: both pieces of a
// half, the same piece of both halves, or one piece.  (Eight copies of 8 KB a slice and block, whose issue paced the loop: 8192 x 2048 998 us; so 962.
// Figures beside this kernel are of single passes; where passes follow one another, the power cap takes 1.1 to 1.2 times as long.)
enum { MAP_HALF = 0, MAP_ACROSS = 1, MAP_PIECE = 2, kMaps = 3 };
struct ProductParams {
    CUtensorMap map[kMaps];
    Common c;
    int* err;
    unsigned long long limit_ns;  // of a wait
    int rounds, tiles;
    int first_class;           // matrices of the first class
    int out_half;              // RESULT is fp16
    bool apply;                // RESULT goes into parameters: p = p keep - rate scale result
    float keep, rate;
};

// A parameter's element with its update.
__device__ __forceinline__ float applied(const ProductParams& P, float param, float v, float rate) { return param * P.keep - rate * v; }
// Results at elements e ... of the output, of which `have` exist.
__device__ __forceinline__ void put1(const ProductParams& P, uint8_t* out, uint8_t* half, long long e, float v, float rate) {
    if (P.apply) {
        float* const p = reinterpret_cast<float*>(out) + e;
        const float next = applied(P, load_global(p), v, rate);
        *p = next;
        if (half) reinterpret_cast<__half*>(half)[e] = __float2half_rn(next);
    } else if (P.out_half) {
        reinterpret_cast<__half*>(out)[e] = __float2half_rn(v);
    } else {
        reinterpret_cast<float*>(out)[e] = v;
    }
}
__device__ __forceinline__ void put4(const ProductParams& P, uint8_t* out, uint8_t* half, long long e, int have, float4 v, float rate) {
    const bool f16 = P.out_half != 0;
    const bool vectors = have >= 4 && (reinterpret_cast<uintptr_t>(out) + e * (f16 ? 2 : 4)) % (f16 ? 8 : 16) == 0 &&
                         (!half || (reinterpret_cast<uintptr_t>(half) + e * 2) % 8 == 0);
    if (!vectors) {
        put1(P, out, half, e, v.x, rate);
        if (have > 1) put1(P, out, half, e + 1, v.y, rate);
        if (have > 2) put1(P, out, half, e + 2, v.z, rate);
        if (have > 3) put1(P, out, half, e + 3, v.w, rate);
        return;
    }
    if (P.apply) {
        const float4 w = load_global(reinterpret_cast<const float4*>(out + e * 4));
        v = make_float4(applied(P, w.x, v.x, rate), applied(P, w.y, v.y, rate), applied(P, w.z, v.z, rate), applied(P, w.w, v.w, rate));
    }
    __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    const uint2 h = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    if (f16) {
        *reinterpret_cast<uint2*>(out + e * 2) = h;
    } else {
        *reinterpret_cast<float4*>(out + e * 4) = v;
        if (half) *reinterpret_cast<uint2*>(half + e * 2) = h;
    }
}


// Two sums in one instruction.
__device__ __forceinline__ void add2(float& a, float& b, uint32_t x, uint32_t y) {
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}" : "+f"(a), "+f"(b) : "r"(x), "r"(y));
}
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
// Registers: a thread of the epilogue holds 128 accumulators beside the eight columns it is splitting.  The block is launched with kLaunchRegs for each thread;
// the four warps of the producer and the MMA give of theirs to the others' (128 x 72 + 256 x 216 = 384 x 168).
constexpr int kLaunchRegs = 168, kControlRegs = 72, kEpilogueRegs = 216;
static_assert(128 * kControlRegs + 32 * kEpilogueWarps * kEpilogueRegs <= kThreads * kLaunchRegs, "more than the block has: the warps that ask for more would wait for good");
// Shared memory, all that a block may have: the ring, and 4 KB for each epilogue warp.
constexpr int kRing = 196608, kStaging = 4096;
constexpr size_t kProductSmem = kRing + kEpilogueWarps * kStaging + 1024;
constexpr int kMaxStages = 6;
constexpr int kQueue = 4;            // tiles that the producer may be ahead

// The tensor core truncates where it adds to an accumulator: about 2^-24 of the sum for each instruction, all to one side (measured: 2.5 x 2^-24 of a
// sum of positive products over K = 64, 98 over 1024).  In three products over K = 8192 that was 7e-5 of the result.  So with two halves the epilogue
// warps take the accumulators of every K slice of 64 and add them in registers, rounded to nearest, while the next slice goes to the other
// accumulators; and within a slice the mixed products come first, while the sums are 2^11 times smaller: four additions count.
// (One product of halves, of 2^-12, does not need it.)

struct Info {        // of a matrix
    int m, n, nb, wide, fine, parts;
    uint32_t x[2], sym, partial;
    float factor;    // of the accumulators, a power of two: from X's scale to that of what is written
};
// Thirty-two rows and columns of a result, from a warp's room in shared memory.
__device__ __forceinline__ void write_columns(const ProductParams& P, const uint8_t* staging, uint8_t* out, uint8_t* half, float rate, long long out_i,
                                           long long out_j, int i0, int m, int j0, int n) {
    const int lane = threadIdx.x & 31;
    if (out_j == 1) {
        const int j = j0 + (lane & 7) * 4, have = n - j;
        if (have <= 0) return;
        if (P.apply && have >= 4 && (reinterpret_cast<uintptr_t>(out) | out_i * 4) % 16 == 0 && (reinterpret_cast<uintptr_t>(half) | out_i * 2) % 8 == 0) {
            // (four loads in flight, from L2: two at a time, and from memory, the parameters' latency was 140 of 1560 us of a step over 34 million of them)
            long long e = (i0 + lane / 8) * out_i + j;
#pragma unroll 1
            for (int q0 = 0; q0 < 8; q0 += 4) {
                float4 w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (i0 + (q0 + q) * 4 + lane / 8 < m) w[q] = load_global(reinterpret_cast<const float4*>(out + (e + q * 4 * out_i) * 4));
#pragma unroll
                for (int q = 0; q < 4; ++q, e += 4 * out_i) {
                    const int r = (q0 + q) * 4 + lane / 8;
                    if (i0 + r >= m) return;
                    const float4 v = *reinterpret_cast<const float4*>(staging + swizzled(r, lane & 7));
                    const float4 next = make_float4(applied(P, w[q].x, v.x, rate), applied(P, w[q].y, v.y, rate), applied(P, w[q].z, v.z, rate), applied(P, w[q].w, v.w, rate));
                    *reinterpret_cast<float4*>(out + e * 4) = next;
                    if (half) {
                        const __half2 a = __floats2half2_rn(next.x, next.y), b = __floats2half2_rn(next.z, next.w);
                        *reinterpret_cast<uint2*>(half + e * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                    }
                }
            }
            return;
        }
#pragma unroll 2
        for (int q = 0; q < 8; ++q) {
            const int r = q * 4 + lane / 8;
            if (i0 + r < m) put4(P, out, half, (i0 + r) * out_i + j, have, *reinterpret_cast<const float4*>(staging + swizzled(r, lane & 7)), rate);
        }
    } else if (i0 + lane < m) {
        long long e = (i0 + lane) * out_i + j0 * out_j;
        if (P.apply && n - j0 >= 32) {
#pragma unroll 1
            for (int q0 = 0; q0 < 32; q0 += 4) {
                float w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = load_global(reinterpret_cast<const float*>(out) + e + q * out_j);
#pragma unroll
                for (int q = 0; q < 4; ++q, e += out_j) {
                    const float next = applied(P, w[q], *reinterpret_cast<const float*>(staging + swizzled(lane, (q0 + q) >> 2) + (q & 3) * 4), rate);
                    reinterpret_cast<float*>(out)[e] = next;
                    if (half) reinterpret_cast<__half*>(half)[e] = __float2half_rn(next);
                }
            }
            return;
        }
#pragma unroll 2
        for (int q = 0; q < min(32, n - j0); ++q, e += out_j)
            put1(P, out, half, e, *reinterpret_cast<const float*>(staging + swizzled(lane, q >> 2) + (q & 3) * 4), rate);
    }
}
// Brings the parameters of a warp's 32 rows and `columns` columns into L2, while the tile's products run.
__device__ __forceinline__ void prefetch_columns(const uint8_t* out, long long out_i, long long out_j, int i0, int m, int j0, int n, int columns) {
    const int lane = threadIdx.x & 31;
    auto fetch = [&](long long e) { asm volatile("prefetch.global.L2 [%0];" ::"l"(__cvta_generic_to_global(out + e * 4))); };
    const int end = min(n, j0 + columns);
    if (i0 >= m) return;
    if (out_j == 1) {
        if (i0 + lane < m)
            for (int j = j0; j < end; j += 32) fetch((i0 + lane) * out_i + j);
    } else {
        for (int j = j0 + lane; j < end; j += 32) fetch(i0 * out_i + j * out_j);
    }
}

// A tile, as the producer passes it on.
struct Tile {
    int k;           // matrix of the group; -1: no more tiles
    int i, j;        // its block row; its (first) block column
    int job;
    int column;      // its first 64-column group in that block: 0 or 1
    int groups;      // 64-column groups of it; 0: none that is in use
    int part, from;  // of K, and its first slice
    int slices;      // of 64 along K; 0: no product
    int extra;       // "f16" update: slices of a I times X's low half behind them
    Info w;
    Op op;
};
constexpr int kOpWords = sizeof(Op) / 4;
static_assert(kOpWords <= 32, "a lane to a word");
__device__ __forceinline__ int claim(int* counter) {
    int v;
    asm volatile("atom.relaxed.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(__cvta_generic_to_global(counter)) : "memory");
    return v;
}
__device__ __forceinline__ int load_acquire(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(__cvta_generic_to_global(p)) : "memory");
    return v;
}
__device__ __forceinline__ void add_release(int* p, int v) {
    asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(__cvta_generic_to_global(p)), "r"(v) : "memory");
}
// What other blocks stored and this thread has acquired is seen by its bulk copies.
__device__ __forceinline__ void fence_proxies() { asm volatile("fence.proxy.async;" ::: "memory"); }

// A lane to a word of the other block's shared memory.
__device__ __forceinline__ void store_remote(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// Tiles of symmetric products: the blocks on and below the diagonal, or, for pairs of block rows, those of both rows up to the lower one's diagonal
// (the upper one's last is above it, and not stored).
template <bool kPair>
__host__ __device__ __forceinline__ int symmetric_count(int mb) {
    const int pairs = (mb + 1) / 2;
    return kPair ? pairs * (pairs + 1) - (mb & 1) : mb * (mb + 1) / 2;
}

// kPair: a cluster of two blocks takes a tile of two block rows with cta_group::2 products, 256 x 128 or 256 x 256.  An SM then holds its own 128 rows and
// half of the columns of a slice, so shared memory, which paces the tiles of one block (a slice of 128 x 128 in three products reads 128 KB and takes
// in 64: 1250 clocks, where the tensor core needs 768; 128 x 256 1875 for 1536), has a quarter (a third) less to deliver, and a stage is as much smaller.
// The first block takes the tiles and passes them to the other one; each loads its own operands, whose arrival the first one's barrier counts, and
// stores its own row.  What the accumulators' readers of the other block tell the first one is a barrier's arrival without a fence: with one, behind
// which the stores of the last tile had to be visible, the pair was slower than two blocks (2048 x 8192 1331 us; without 970; two blocks then 1197).
template <int kPlanes, bool kPair>
__global__ void __launch_bounds__(kThreads, 1) ortho_product_kernel(const __grid_constant__ ProductParams P) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], tfull_bar[4], tempty_bar[4], qfull_bar[kQueue], qempty_bar[kQueue],
        drain_bar;
    __shared__ __align__(8) int abort_state[4];
    __shared__ uint32_t tmem_base;
    __shared__ int first[4][kGroup];  // of X X^T, symmetric products, Q X, SUM
    __shared__ __align__(16) Tile queue[kQueue];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    volatile int* const abort_flag = abort_state;
    // A stage holds a K slice of both operands: 128 rows of the left one and 128 columns (symmetric products) or 256 (X) of the right one, of a pair
    // half of them in each block.
    constexpr uint32_t kNarrowB = kPair ? kPiece : kHalf, kWideB = kPair ? kHalf : 2 * kHalf;  // of a plane of the right one
    constexpr uint32_t kNarrow = kPlanes * (kHalf + kNarrowB), kWideStage = kPlanes * (kHalf + kWideB);
    constexpr int kBoth = kPair ? 2 : 1, kReports = kBoth * kEpilogueWarps;
    const uint32_t rank = kPair ? nml::cluster_ctarank() : 0;
    const bool leader = rank == 0;

    if (warp == 0) {
        if (kPair) nml::tmem_alloc_pair(nml::smem_u32(&tmem_base), 512); else nml::tmem_alloc(nml::smem_u32(&tmem_base), 512);
    }
    if (tid == 32) {
        for (int s = 0; s < kMaxStages; ++s) {
            nml::mbar_init(nml::smem_u32(&full_bar[s]), 1);  // (of a pair the first block's counts both blocks' copies)
            nml::mbar_init(nml::smem_u32(&empty_bar[s]), 1);
        }
        for (int b = 0; b < 4; ++b) {
            nml::mbar_init(nml::smem_u32(&tfull_bar[b]), 1);
            nml::mbar_init(nml::smem_u32(&tempty_bar[b]), kReports);
        }
        for (int q = 0; q < kQueue; ++q) {
            nml::mbar_init(nml::smem_u32(&qfull_bar[q]), 1);
            nml::mbar_init(nml::smem_u32(&qempty_bar[q]), (kPair && leader ? 2 : 1) + kEpilogueWarps);  // (the other block's users are one)
        }
        nml::mbar_init(nml::smem_u32(&drain_bar), 1);
        nml::fence_mbar_init();
        nml::abort_state_init(abort_flag, P.limit_ns);
    }
    pdl_enter();
    const bool skip = skipped(P.c.skip);
    const int count = P.c.count;
    for (int i = tid; i < count; i += kThreads) {
        first[0][i] = load_global(&P.c.table[i].first_gram);
        first[1][i] = load_global(&P.c.table[i].first_symmetric);
        first[2][i] = load_global(&P.c.table[i].first_update);
        first[3][i] = load_global(&P.c.table[i].first_parts);
    }
    nml::tc_fence_before();
    __syncthreads();
    if (kPair) nml::cluster_sync_all();  // (barriers are there before the other block arrives on them)
    nml::tc_fence_after();
    const uint32_t tmem = tmem_base;
    auto symmetric_first = [&](const Info& w, int buffer) { return w.sym + buffer * lower((w.m + kBlock - 1) / kBlock, 0); };
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, nml::mbar_wait(nml::smem_u32(bar), parity, abort_flag, P.err, code)) != 0;
    };
    // for what the other block of a pair has arrived with
    auto wait_other = [&](uint64_t* bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, nml::mbar_wait<false, kPair>(nml::smem_u32(bar), parity, abort_flag, P.err, code)) != 0;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == 0) {
            // ------------------------------------------------------------ producer: takes tiles, then a lane to a copy of 8 KB
            const int tiles = skip ? 0 : P.tiles;
            const Round* const rounds = P.c.rounds;
            int slot = 0, s = 0, stages = 0;
            uint32_t qparity = 0, parity = 0, used = 0;  // bits of parity: phase of each stage's next use; of used: stages not known to be free
            uint32_t now_stage = 0;
            bool ok = true;
            int round = 0;
            int next_first = tiles ? load_global(&rounds[min(1, P.rounds - 1)].first) : 0;
            while (ok) {
                Tile tile;
                Info w;
                int mb, symmetric_tiles, per_row, whole;
                bool is_wide;
                const int now = slot;
                if (leader) {
                    // (not before the last tile's copies are issued: a block that held a second tile of a product would make that product twice as long)
                    int t = 0;
                    if (lane == 0) t = claim(P.c.done);
                    t = __shfl_sync(0xffffffffu, t, 0);
                    tile.k = -1;
                    if (t < tiles) {
                        while (round + 1 < P.rounds && t >= next_first) {
                            ++round;
                            next_first = load_global(&rounds[min(round + 1, P.rounds - 1)].first);
                        }
                        t -= load_global(&rounds[round].first);
                        const int of_first = load_global(&rounds[round].of_first), cls = t >= of_first;
                        if (cls) t -= of_first;
                        const int* const words = reinterpret_cast<const int*>(&rounds[round].op[cls]);
                        const int word = lane < kOpWords ? load_global(words + lane) : 0;
                        const int kind = __shfl_sync(0xffffffffu, word, offsetof(Op, kind) / 4), jobs = __shfl_sync(0xffffffffu, word, offsetof(Op, jobs) / 4);
                        const int gram = __shfl_sync(0xffffffffu, word, offsetof(Op, gram) / 4), grown = __shfl_sync(0xffffffffu, word, offsetof(Op, grown) / 4);
                        is_wide = kind == ITERATE || kind == RESULT;
                        whole = kind == POLY && gram;
                        // (matrices of the first class come first, and their tiles count from 0; those of the second behind all of the first)
                        const int n0 = P.first_class;
                        const int lo = cls ? n0 : 0, hi = cls ? count : n0;
                        const int* const starts = first[is_wide ? 2 : kind == SUM ? 3 : whole ? 0 : 1];
                        const int base = starts[lo], per_job = is_wide ? 1 : jobs;
                        int a = lo, b = hi - 1;
                        while (a < b) {
                            const int mid = (a + b + 1) / 2;
                            if ((starts[mid] - base) * per_job <= t) a = mid; else b = mid - 1;
                        }
                        tile.k = a;
                        t -= (starts[a] - base) * per_job;
                        {
                            const Work* const from = P.c.table + a;
                            auto word = [](const uint32_t* p) { return static_cast<uint32_t>(load_global(reinterpret_cast<const int*>(p))); };
                            w = {load_global(&from->s.m), load_global(&from->s.n), load_global(&from->nb), load_global(&from->wide), load_global(&from->fine),
                                 load_global(&from->parts), {word(&from->x[0]), word(&from->x[1])}, word(&from->sym), word(&from->partial), 1.f};
                            const int lift = load_global(&from->lift), scale = load_global(&from->sx) + lifted(lift, grown & ((1 << kGrownBits) - 1));
                            if (gram) w.factor = power_of_two(-2 * scale);
                            if (kind == RESULT) w.factor = power_of_two(-scale);
                            if (kind == ITERATE) w.factor = power_of_two(lifted(lift, grown >> kGrownBits) - lifted(lift, grown & ((1 << kGrownBits) - 1)));
                        }
                        mb = (w.m + kBlock - 1) / kBlock;
                        symmetric_tiles = symmetric_count<kPair>(mb) * w.fine;
                        const int wide_groups = (w.n + 63) / 64;
                        per_row = (wide_groups + w.wide - 1) / w.wide;
                        tile.extra = tile.job = tile.column = tile.part = tile.from = 0;
                        if (is_wide) {
                            tile.i = t / per_row;
                            const int group = t % per_row * w.wide;
                            tile.j = group >> 1;
                            tile.column = group & 1;
                            tile.groups = min(w.wide, wide_groups - group);
                            tile.slices = (w.m + 63) / 64;
                            if (kPlanes == 1) tile.extra = min(2, tile.slices - 2 * tile.i);
                        } else {
                            const int fine = kind == SUM ? 2 : w.fine;
                            if (whole) {
                                tile.part = t / symmetric_tiles;
                                t %= symmetric_tiles;
                            } else if (kind != SUM && t >= symmetric_tiles) {
                                t -= symmetric_tiles;
                                tile.job = 1;
                            }
                            if (fine == 2) {
                                tile.column = t & 1;
                                t >>= 1;
                            }
                            // the row: of row i there are i (i + 1) / 2 tiles in front, of pair i twice as many
                            auto in_front = [](int i) { return kBoth * (i * (i + 1) / 2); };
                            tile.i = static_cast<int>((sqrtf(8.f / kBoth * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
                            while (in_front(tile.i) > t) --tile.i;
                            while (in_front(tile.i + 1) <= t) ++tile.i;
                            tile.j = t - in_front(tile.i);
                            tile.groups = max(0, min(3 - fine, (w.m - tile.j * kBlock + 63) / 64 - tile.column));
                            const int all = ((whole ? w.n : w.m) + 63) / 64, share = whole ? (all + w.parts - 1) / w.parts : all;
                            tile.from = tile.part * share;
                            tile.slices = kind == SUM || tile.groups == 0 ? 0 : min(share, all - tile.from);
                        }
                        // pass it on
                        if (!wait_other(&qempty_bar[slot], qparity ^ 1, nml::ERR_WAIT_EMPTY)) {
                            ok = false;
                            break;
                        }
                        if (lane < kOpWords) reinterpret_cast<int*>(&queue[slot].op)[lane] = word;
                        if (lane == 0) {
                            queue[slot].k = tile.k, queue[slot].i = tile.i, queue[slot].j = tile.j, queue[slot].job = tile.job, queue[slot].column = tile.column;
                            queue[slot].groups = tile.groups, queue[slot].part = tile.part, queue[slot].from = tile.from, queue[slot].slices = tile.slices, queue[slot].extra = tile.extra;
                            queue[slot].w = w;
                        }
                        __syncwarp();
                    } else {
                        if (!wait_other(&qempty_bar[slot], qparity ^ 1, nml::ERR_WAIT_EMPTY)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) queue[slot].k = -1;
                        __syncwarp();
                    }
                    if (kPair) {  // to the other block
                        const uint32_t to = nml::map_to_cta(nml::smem_u32(&queue[slot]), 1);
                        const uint32_t* const words = reinterpret_cast<const uint32_t*>(&queue[slot]);
                        for (int e = lane; e < static_cast<int>(sizeof(Tile) / 4); e += 32) store_remote(to + 4 * e, words[e]);
                        __syncwarp();
                    }
                } else {
                    if (!wait_other(&qfull_bar[slot], qparity, nml::ERR_WAIT_FULL)) {
                        ok = false;
                        break;
                    }
                    tile = queue[slot];
                    if (tile.k < 0) break;
                    w = tile.w;
                    is_wide = tile.op.kind == ITERATE || tile.op.kind == RESULT;
                    whole = tile.op.kind == POLY && tile.op.gram;
                    mb = (w.m + kBlock - 1) / kBlock;
                    symmetric_tiles = symmetric_count<kPair>(mb) * w.fine;
                    per_row = ((w.n + 63) / 64 + w.wide - 1) / w.wide;
                }
                const Op& op = queue[now].op;  // (the producer's own copy stays until it comes round to the slot again; the other block's until it is given back)
                // the matrix's earlier products: to be waited for before its copies are issued, or, where there are none, before it is passed on
                auto wait_for_matrix = [&](const Op& op) {
                    const int need = kReports * (op.gram_before * symmetric_tiles * w.parts + op.symmetric_before * symmetric_tiles +
                                                       op.wide_before * ((mb + kBoth - 1) / kBoth) * per_row + op.sum_before * (w.parts > 1 ? 2 * lower(mb, 0) : 0));
                    if (need == 0) return true;
                    int gave_up = 0;
                    if (lane == 0) {
                        const int* const done = P.c.done + 1 + tile.k;
                        uint64_t t0 = 0;
                        for (uint32_t it = 1; load_acquire(done) < need; ++it) {
                            __nanosleep(40);
                            if ((it & 0xff) != 0) continue;
                            const uint64_t now = nml::globaltimer_ns();
                            if (t0 == 0) t0 = now;
                            if (*abort_flag || now - t0 > *reinterpret_cast<volatile unsigned long long*>(abort_flag + 2)) {
                                *abort_flag = 1;
                                atomicCAS(P.err, 0, nml::ERR_WAIT_TILES);
                                gave_up = 1;
                                break;
                            }
                        }
                    }
                    if (__shfl_sync(0xffffffffu, gave_up, 0)) return false;
                    fence_proxies();
                    return true;
                };
                if (leader) {
                    if (tile.k >= 0 && tile.slices == 0 && !wait_for_matrix(op)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        nml::mbar_arrive(nml::smem_u32(&qfull_bar[now]));
                        if (kPair) nml::mbar_arrive_cluster(nml::map_to_cta(nml::smem_u32(&qfull_bar[now]), 1));
                    }
                }
                if (++slot == kQueue) slot = 0, qparity ^= 1;
                if (tile.k < 0) break;
                if (tile.slices > 0) {
                    if (!wait_for_matrix(op)) {
                        ok = false;
                        break;
                    }
                    // its K slices; a ring of stages of the other size only begins when the last one's are free
                    const uint32_t stage_bytes = is_wide ? kWideStage : kNarrow, b_bytes = is_wide ? kWideB : kNarrowB;
                    if (now_stage != stage_bytes) {
                        for (int e = 0; ok && e < stages; ++e)
                            if (used >> e & 1) ok = wait(&empty_bar[e], (parity >> e & 1) ^ 1, nml::ERR_WAIT_EMPTY);
                        if (!ok) break;
                        used = 0;
                        s = 0;
                        now_stage = stage_bytes;
                        stages = min(kMaxStages, static_cast<int>(kRing / stage_bytes));
                    }
                    const bool same = whole && tile.i == tile.j;
                    const int b_pieces = same ? 0 : tile.groups, pieces = kPlanes * (2 + b_pieces);
                    const bool is_a = lane < (kPair ? 1 : 2 * kPlanes);
                    const int at = is_a ? lane : lane - 2 * kPlanes, per = is_a ? 2 : max(1, b_pieces);
                    const int plane = at / per, piece = at % per;
                    const uint32_t dst = kPair ? (is_a ? 0 : kPlanes * kHalf) : (is_a ? plane * kHalf : kPlanes * kHalf + plane * b_bytes) + piece * kPiece;
                    const uint32_t buffer = symmetric_first(w, is_wide ? op.left : is_a ? op.job[tile.job].left : op.job[tile.job].right);
                    const uint32_t x = op.from ? w.x[1] : w.x[0];
                    // block row of the left operand; a pair that is one row short has its last one twice.  K-major up to `turn`, for both rows alike
                    const int left_row = min(kBoth * tile.i + static_cast<int>(rank), mb - 1), turn = is_a ? kBoth * tile.i : tile.j;
                    const int right_block = min(tile.j + static_cast<int>(rank), w.nb - 1);
                    for (int q = 0; q < tile.slices + tile.extra; ++q) {
                        if (used >> s & 1) {
                            if (!wait(&empty_bar[s], (parity >> s & 1) ^ 1, nml::ERR_WAIT_EMPTY)) {
                                ok = false;
                                break;
                            }
                        }
                        const uint32_t bar = nml::smem_u32(&full_bar[s]), to = nml::smem_u32(smem) + s * stage_bytes + dst;
                        if (lane == 0 && leader) nml::mbar_arrive_expect_tx(bar, kPair ? 2 * stage_bytes : pieces * kPiece);
                        __syncwarp();
                        if (kPair && lane < 2) {  // a lane to an operand
                            const int kq = tile.from + q, kb = kq >> 1, h = kq & 1;
                            const bool own = lane == 0, both = own || is_wide;  // the left operand; both pieces of the right one
                            const int row = own ? left_row : tile.j;
                            bool straight = true;
                            int block;
                            if (whole) {
                                block = static_cast<int>(x) + row * w.nb + kb;
                            } else if (!own && is_wide) {
                                block = static_cast<int>(x) + kb * w.nb + right_block;
                                straight = false;
                            } else {
                                straight = kb <= turn;
                                block = static_cast<int>(buffer) + (straight ? lower(row, kb) : lower(kb, row));
                            }
                            const int mine = both ? 0 : static_cast<int>(rank);
                            nml::tma_load_5d_pair(to, &P.map[both ? (straight ? MAP_HALF : MAP_ACROSS) : MAP_PIECE], nml::map_to_cta(bar, 0), 0, 0, straight ? mine : h,
                                                  straight ? h : mine, 2 * block);
                        }
                        if (!kPair && lane < pieces) {
                            const bool low = q >= tile.slices;  // a I times X's low half
                            const int kq = low ? 2 * tile.i + q - tile.slices : tile.from + q, kb = kq >> 1, h = kq & 1;
                            const int group = is_a ? piece : piece + tile.column;
                            const uint8_t* from;
                            const uint32_t straight = (h * 2 + group) * kPiece, across = (group * 2 + h) * kPiece;  // K-major; MN-major
                            auto symmetric = [&](int row) {
                                return kb <= turn ? block_at(P.c.blocks, buffer, lower(row, kb)) + straight : block_at(P.c.blocks, buffer, lower(kb, row)) + across;
                            };
                            if (!is_wide) {
                                const int row = is_a ? left_row : tile.j;
                                from = whole ? block_at(P.c.blocks, x, row * w.nb + kb) + straight : symmetric(row);
                            } else if (is_a) {
                                from = low ? block_at(P.c.blocks, op.identity, 0) + straight : symmetric(left_row);
                            } else {  // X's rows along K: two 64-column groups to a block
                                from = block_at(P.c.blocks, x, kb * w.nb + tile.j + (group >> 1)) + (low ? kPlane : 0) + ((group & 1) * 2 + h) * kPiece;
                            }
                            from += plane * kPlane;
                            nml::bulk_load(to, from, kPiece, bar);
                        }
                        __syncwarp();
                        used |= 1u << s;
                        parity ^= 1u << s;
                        if (++s == stages) s = 0;
                    }
                }
                if (!ok) break;
                if (kPair && !leader) {
                    __syncwarp();
                    if (lane == 0) nml::mbar_arrive(nml::smem_u32(&qempty_bar[now]));
                }
            }
            if (leader && (!ok || *abort_flag)) {  // no copy may be in flight when the block's shared memory goes away
                for (int e = 0; e < stages; ++e) {
                    if (!(used >> e & 1)) continue;
                    const uint64_t t0 = nml::globaltimer_ns();
                    while (!nml::mbar_try_wait(nml::smem_u32(&full_bar[e]), (parity >> e & 1) ^ 1)) {
                        if (nml::globaltimer_ns() - t0 > 2000000ull) {
                            if (lane == 0) atomicCAS(P.err, 0, nml::ERR_WAIT_DRAIN);
                            break;
                        }
                    }
                }
            }
        } else if (kPair && warp == 1 && !leader) {
            // ------------------------------------------------------------ tells the first block which tiles this one is through with
            int slot = 0;
            uint32_t qparity = 0;
            while (true) {
                if (!wait_other(&qfull_bar[slot], qparity, nml::ERR_WAIT_FULL) || queue[slot].k < 0) break;
                if (!wait(&qempty_bar[slot], qparity, nml::ERR_WAIT_EMPTY)) break;
                if (lane == 0) nml::mbar_arrive_cluster(nml::map_to_cta(nml::smem_u32(&qempty_bar[slot]), 0));
                __syncwarp();
                if (++slot == kQueue) slot = 0, qparity ^= 1;
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA
            int slot = 0, s = 0, stages = 0, unit = 0;
            uint32_t qparity = 0, parity = 0, tparity = 0, pairs = 0, now_stage = 0;  // pairs: of units whose last use was by both
            bool ok = true;
            const uint32_t ring = nml::smem_u32(smem);
            auto commit = [&](uint64_t* bar) {  // (of a pair in both blocks)
                if (kPair) nml::umma_commit_pair(nml::smem_u32(bar)); else nml::umma_commit(nml::smem_u32(bar));
            };
            while (ok) {
                if (!wait(&qfull_bar[slot], qparity, nml::ERR_WAIT_FULL)) {
                    ok = false;
                    break;
                }
                const int k = queue[slot].k, row = queue[slot].i, column = queue[slot].j, groups = queue[slot].groups, real = queue[slot].slices;
                const int slices = real + queue[slot].extra, kind = queue[slot].op.kind, in_block = queue[slot].column;
                const bool is_wide = kind == ITERATE || kind == RESULT, gram = queue[slot].op.gram != 0;
                if (k < 0) break;
                __syncwarp();
                if (lane == 0) nml::mbar_arrive(nml::smem_u32(&qempty_bar[slot]));
                if (++slot == kQueue) slot = 0, qparity ^= 1;
                if (slices == 0) continue;
                const uint32_t stage_bytes = is_wide ? kWideStage : kNarrow, b_bytes = is_wide ? kWideB : kNarrowB;
                if (now_stage != stage_bytes) {
                    s = 0;
                    now_stage = stage_bytes;
                    stages = min(kMaxStages, static_cast<int>(kRing / stage_bytes));
                }
                const bool same = !kPair && gram && row == column;
                for (int q = 0; q < slices; ++q) {
                    if (kPlanes == 2 || q == 0) {
                        // TMEM is four units of 128 columns, each with its barriers; a wide tile takes two, and the first one's barriers
                        if (is_wide && (unit & 1)) unit = (unit + 1) & 3;
                        const int pair = unit >> 1;
                        auto drained = [&](int u) { return wait(&tempty_bar[u], (tparity >> u & 1) ^ 1, nml::ERR_WAIT_TMEM_EMPTY); };
                        ok = drained(unit) && (!is_wide || drained(unit + 1)) && (is_wide || !(unit & 1) || !(pairs >> pair & 1) || drained(unit - 1));
                        if (!ok) break;
                        if (is_wide) pairs |= 1u << pair; else pairs &= ~(1u << pair);
                        nml::tc_fence_after();
                    }
                    if (!wait(&full_bar[s], parity >> s & 1, nml::ERR_WAIT_FULL)) {
                        ok = false;
                        break;
                    }
                    nml::tc_fence_after();
                    const bool low = q >= real, last = kPlanes == 2 || q + 1 == slices;
                    const int kb = q >> 1;
                    const int a_mn = !gram && !low && kb > kBoth * row;
                    const int b_mn = is_wide ? 1 : !gram && kb > column;
                    const uint32_t idesc = nml::make_instr_desc(0, a_mn, b_mn, kBoth * 128, kPair ? (is_wide ? 256 : 128) : groups * 64);
                    const uint32_t sa = ring + s * stage_bytes, sb = same ? sa + in_block * kPiece : sa + kPlanes * kHalf, bp = same ? kHalf : b_bytes;
                    if (nml::elect_one()) {
                        const uint64_t a0 = nml::make_smem_desc(sa, kPiece, 1024, 2), b0 = nml::make_smem_desc(sb, kPiece, 1024, 2);
                        const uint32_t a_step = (a_mn ? 2048 : 32) >> 4, b_step = (b_mn ? 2048 : 32) >> 4;
#pragma unroll
                        for (int p = kPlanes == 2 ? 2 : 0; p >= 0; --p) {  // low x high, high x low, high x high
                            uint64_t ad = a0 + (p == 2 ? kHalf >> 4 : 0), bd = b0 + (p == 1 ? bp >> 4 : 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e, ad += a_step, bd += b_step) {
                                const bool add = kPlanes == 2 ? e > 0 || p < 2 : e > 0 || q > 0;
                                if (kPair) nml::umma_f16_pair(tmem + unit * 128, ad, bd, idesc, add); else nml::umma_f16(tmem + unit * 128, ad, bd, idesc, add);
                            }
                        }
                        commit(&empty_bar[s]);
                        if (last) commit(&tfull_bar[unit]);
                    }
                    __syncwarp();
                    parity ^= 1u << s;
                    if (++s == stages) s = 0;
                    if (last) {
                        tparity ^= 1u << unit;
                        unit = (unit + (is_wide ? 2 : 1)) & 3;
                    }
                }
            }
            if (!ok) {  // the products issued so far still read shared memory and write TMEM
                if (nml::elect_one()) commit(&drain_bar);
                __syncwarp();
                const uint64_t t0 = nml::globaltimer_ns();
                while (!nml::mbar_try_wait(nml::smem_u32(&drain_bar), 0)) {
                    if (nml::globaltimer_ns() - t0 > 2000000ull) {
                        if (lane == 0) atomicCAS(P.err, 0, nml::ERR_WAIT_DRAIN);
                        break;
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
        // ------------------------------------------------------------ epilogue: a thread to a row and half of the columns of the tile
        int slot = 0, unit = 0, pending = -1;  // pending: matrix of a tile that is stored but not reported
        uint32_t qparity = 0, tparity = 0;
        const int quarter = warp & 3, row = quarter * 32 + lane, side = (warp - 4) >> 2;
        uint8_t* const staging = smem + kRing + (warp - 4) * kStaging;
        // A tile is reported when its stores are visible, which takes a while: where the next one is there already, its first slice comes first.
        auto report = [&]() {
            if (pending >= 0) {
                __syncwarp();
                if (lane == 0) add_release(P.c.done + 1 + pending, 1);
                pending = -1;
            }
        };
        while (true) {
            if (!__all_sync(0xffffffffu, nml::mbar_test(nml::smem_u32(&qfull_bar[slot]), qparity))) report();
            if (!wait_other(&qfull_bar[slot], qparity, nml::ERR_WAIT_FULL)) break;
            const int k = queue[slot].k, tile_i = kBoth * queue[slot].i + static_cast<int>(rank), tile_j = queue[slot].j, groups = queue[slot].groups, slices = queue[slot].slices;
            const int in_block = queue[slot].column, part = queue[slot].part;
            const int kind = queue[slot].op.kind, gram = queue[slot].op.gram, from_x = queue[slot].op.from;
            const Symmetric job = queue[slot].op.job[queue[slot].job];
            const float op_f1 = queue[slot].op.f1, op_d1 = queue[slot].op.d1;
            const Info w = queue[slot].w;
            if (k < 0) break;
            __syncwarp();
            if (lane == 0) nml::mbar_arrive(nml::smem_u32(&qempty_bar[slot]));
            if (++slot == kQueue) slot = 0, qparity ^= 1;
            const int mine = groups * 2, g0 = side * mine + 4 * in_block;  // this thread's columns in sixteens; the first one in its block
            const int chunks = kPlanes == 2 ? slices : min(1, slices);
            const bool is_wide = kind == ITERATE || kind == RESULT;
            if (kind == RESULT && P.apply) {
                const Source* src = &P.c.table[k].s;
                prefetch_columns(reinterpret_cast<const uint8_t*>(load_wide(reinterpret_cast<const long long*>(&src->out))), load_wide(&src->out_i), load_wide(&src->out_j),
                                 tile_i * kBlock + quarter * 32, w.m, tile_j * kBlock + g0 * 16, w.n, mine * 16);
            }
            float acc[8][16];
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[c][e] = 0.f;
            bool ok = true;
            for (int q = 0; q < chunks; ++q) {
                if (is_wide && (unit & 1)) unit = (unit + 1) & 3;
                if (q == 0 && !__all_sync(0xffffffffu, nml::mbar_test(nml::smem_u32(&tfull_bar[unit]), tparity >> unit & 1))) report();
                if (!wait(&tfull_bar[unit], tparity >> unit & 1, nml::ERR_WAIT_TMEM_FULL)) {
                    ok = false;
                    break;
                }
                nml::tc_fence_after();
                const uint32_t from = tmem + unit * 128 + side * mine * 16 + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < 8; c += 2) {
                    if (c < mine) {
                        uint32_t r[32];
                        nml::tmem_ld_32x32(from + c * 16, r);
                        nml::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e += 2) add2(acc[c + e / 16][e % 16], acc[c + e / 16][e % 16 + 1], r[e], r[e + 1]);
                    }
                }
                nml::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kPair) nml::mbar_arrive_remote(nml::map_to_cta(nml::smem_u32(&tempty_bar[unit]), 0));
                    else nml::mbar_arrive(nml::smem_u32(&tempty_bar[unit]));
                }
                tparity ^= 1u << unit;
                unit = (unit + (is_wide ? 2 : 1)) & 3;
            }
            if (!ok) break;
            report();
            if (kind == RESULT) {
                const Source* src = &P.c.table[k].s;
                const long long out_i = load_wide(&src->out_i), out_j = load_wide(&src->out_j);
                uint8_t* const out = reinterpret_cast<uint8_t*>(load_wide(reinterpret_cast<const long long*>(&src->out)));
                uint8_t* const half = reinterpret_cast<uint8_t*>(load_wide(reinterpret_cast<const long long*>(&src->half)));
                const float f0 = op_f1 * w.factor, rate = P.rate * load_global(&src->scale);  // (a power of two)
                const int i0 = tile_i * kBlock + quarter * 32, j0 = tile_j * kBlock + g0 * 16;
                // Thirty-two columns at a time go through shared memory: where rows lie densely, eight lanes write a row's 128 bytes; else the lanes
                // of a warp lie beside one another along a column.
#pragma unroll
                for (int c = 0; c < 8; c += 2) {
                    if (c < mine) {
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            *reinterpret_cast<float4*>(staging + swizzled(lane, q)) =
                                make_float4(acc[c + q / 4][q % 4 * 4] * f0, acc[c + q / 4][q % 4 * 4 + 1] * f0, acc[c + q / 4][q % 4 * 4 + 2] * f0,
                                            acc[c + q / 4][q % 4 * 4 + 3] * f0);
                        __syncwarp();
                        write_columns(P, staging, out, half, rate, out_i, out_j, i0, w.m, j0 + c * 16, w.n);
                    }
                }
            } else {
                const bool iterate = kind == ITERATE;
                const uint32_t to = iterate ? (from_x ? w.x[0] : w.x[1]) : symmetric_first(w, job.out);
                const int block = iterate ? tile_i * w.nb + tile_j : lower(tile_i, tile_j);
                // Thirty-two columns of both planes at a time go through shared memory, so that four lanes write 64 contiguous bytes of a row (a thread's
                // own 32 bytes, in 32 lines a store, took 1.1 us a matrix and tile; bulk copies of 4 KB out of shared memory, whose room
                // has to be waited for, 3).
                auto store = [&](uint32_t base, bool low) {
#pragma unroll
                    for (int c = 0; c < 8; c += 2) {
                        if (c < mine) {
                            const int half = (g0 + c) >> 2, part = (g0 + c) >> 1 & 1;
                            uint8_t* const at = block_at(P.c.blocks, base, block + (half >> 1)) + (half & 1) * kHalf + quarter * 4096;
                            __syncwarp();
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint4 h, l;
                                split8(&acc[c + q / 2][q % 2 * 8], h, l);
                                uint8_t* const mine_at = staging + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4);
                                *reinterpret_cast<uint4*>(mine_at) = h;
                                if (low) *reinterpret_cast<uint4*>(mine_at + 2048) = l;
                            }
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int r = e * 8 + (lane >> 2), q = lane & 3;
                                const uint8_t* const from = staging + r * 64 + ((q ^ (r >> 1 & 3)) << 4);
                                uint8_t* const out = at + swizzled(r, part * 4 + q);
                                *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(from);
                                if (low) *reinterpret_cast<uint4*>(out + kPlane) = *reinterpret_cast<const uint4*>(from + 2048);
                            }
                        }
                    }
                };
                auto scale = [&](float f) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[c][e] *= f;
                };
                auto add_diagonal = [&](float d) {  // (symmetric tiles: at most 64 columns to a thread)
                    if (tile_i == tile_j)
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[c][e] += c * 16 + e == row - g0 * 16 ? d : 0.f;
                };
                // (of a last block of 64 rows or fewer, half is never read: K slices and columns end at a multiple of 64, and what the other rows of an
                // operand hold, which may be anything, ends in rows and columns that are not stored either)
                const bool in_use = tile_i * kBlock + (quarter & 2) * 32 < w.m;
                // X X^T in several parts of K: the sums go to memory as they are, [sixteen columns][four of them][row], and come from there in order
                const int mb = (w.m + kBlock - 1) / kBlock;
                const bool partial = kind == POLY && gram && w.parts > 1;
                if (partial && in_use) {
                    float4* const out = reinterpret_cast<float4*>(block_at(P.c.blocks, w.partial, part * lower(mb, 0) + block));
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (c < mine)
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                out[((g0 + c) * 4 + q) * kBlock + row] = make_float4(acc[c][4 * q], acc[c][4 * q + 1], acc[c][4 * q + 2], acc[c][4 * q + 3]);
                }
                if (kind == SUM && in_use) {
                    const float4* const from = reinterpret_cast<const float4*>(block_at(P.c.blocks, w.partial, block));
                    const size_t step = static_cast<size_t>(lower(mb, 0)) * (2 * kPlane / sizeof(float4));
#pragma unroll 2
                    for (int p = 0; p < w.parts; ++p)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            if (c < mine)
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const float4 v = load_shared_by_blocks(from + p * step + ((g0 + c) * 4 + q) * kBlock + row);
                                    acc[c][4 * q] += v.x, acc[c][4 * q + 1] += v.y, acc[c][4 * q + 2] += v.z, acc[c][4 * q + 3] += v.w;
                                }
                }
                const bool above = kPair && !iterate && tile_j > tile_i;  // the diagonal
                const int matrices = !in_use || above || partial || groups == 0 ? 0 : kind == POLY || kind == SUM ? 2 : 1;
#pragma unroll 1
                for (int e = 0; e < matrices; ++e) {  // (A and P: f0 is a power of two)
                    scale(e ? op_f1 / job.f0 : (iterate ? op_f1 : job.f0) * w.factor);
                    if (e || kind == PLAIN) add_diagonal(e ? op_d1 : job.d1);
                    store(e ? symmetric_first(w, kPoly) : to, iterate || kPlanes == 2);
                }
                pending = k;
            }
        }
        report();
    }
    nml::tc_fence_before();
    __syncthreads();
    if (kPair) nml::cluster_sync_all();  // (neither block leaves while the other may still reach it)
    nml::tc_fence_after();
    if (warp == 0) {
        if (kPair) {
            nml::tmem_relinquish_pair();
            nml::tmem_dealloc_pair(tmem, 512);
        } else {
            nml::tmem_relinquish();
            nml::tmem_dealloc(tmem, 512);
        }
    }
}

}  // namespace nml_ortho
#include "nml_ortho_small.cuh"
namespace nml_ortho {

// ---------------------------------------------------------------- parameters that are no matrices --
constexpr int kVectors = 128;          // pieces of one launch
constexpr int kVectorPiece = 16384;    // values of a piece: a longer vector is several
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
// Plain momentum: p = p keep - rate u, a block to a piece of a vector.
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
// a matrix 150 times as large.  (Against 64 bits: 3 + 2 over gradients of five kinds 1e-6 to 8e-6; random 256 x 513 8.0e-6, 400 x 5000 1.4e-5 and 2048 x 8192 1.8e-6, the same
// steps in fp32 2.1e-6, 5.3e-6 and 5.3e-6; all five in one chain 1e-6 to 4e-4.)  "f16" has no such reserve and takes single steps.
constexpr double kGrowth = 150.0;
struct Step {
    double a, b, c;
    int ea, ep, eu, et, eq;  // A, P, U, T and Q are stored times 2^e
    bool starts, ends;       // a chain
    int grown;               // where it ends: log2 of what X may have been multiplied by, at least 0
    double amplified;        // an error of the Gram matrix by this step, at most
};
struct Polynomial {
    Step step[kMaxSteps];
    int steps = 0;
    double largest = 1.0;    // singular value at the chains' starts, hence element of X
};
static int exponent_below(double bound) {  // largest e with bound * 2^e <= 2^15
    return std::max(-24, std::min(24, static_cast<int>(floor(log2(32768.0 / std::max(bound, 1e-6))))));
}
static bool polynomial(const double* coefficients, int steps, bool chained, Polynomial* p) {
    constexpr int kPoints = 128;        // singular values, at which the matrices' eigenvalues are followed
    constexpr double kBetween = 1.01;   // and what lies between two of them
    double l = kBetween, lambda[kPoints + 1], q[kPoints + 1], growth = 1.0, multiplied = 0.0;  // (log2)
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
        s.amplified = std::max(1.0, mu * mu);
        growth *= s.amplified;
        if (!(next <= 4096.0)) return false;  // singular values beyond 64
        s.ends = !chained || k == steps - 1 || growth > kGrowth;
        starts = s.ends;
        if (s.ends) {
            l = std::max(sqrt(next) * kBetween, 1e-3), p->largest = std::max(p->largest, l);
            multiplied += log2(std::max(mq * kBetween, 1e-30));
            s.grown = std::max(0, std::min(kMostLift, static_cast<int>(ceil(multiplied))));
        }
    }
    return true;
}

// Which matrices are chained: where the long side is so much longer that products of m x m matrices are the cheaper ones, and m is so large that
// the rounding errors, which are random, add to little in any one direction (relative to fp32 products, errors were 2.0 at m = 256, 7 at 64).  1024 x
// 4096 412 us instead of 463, eight of them 1051 / 1612, 256 x 1024 190 / 201; 512 x 768 231 / 221, 1024 x 1024 would be 340 / 307, 512 x 512 223 / 203.
static bool chained(const Source& s, int math) { return math == NML_MATH_3XF16 && s.m >= 256 && 2ll * s.n >= 3ll * s.m; }

struct Plan {
    int sums = 0, halves = 0, first_class = 0;
    int gram_tiles[kClasses] = {0, 0}, symmetric_tiles[kClasses] = {0, 0}, update_tiles[kClasses] = {0, 0}, sum_tiles[kClasses] = {0, 0};
    uint32_t blocks = 0, identity = 0;
    bool pair = false;
    size_t sums_at = 0, rounds_at = 0, done_at = 0, blocks_at = 0, bytes = 0;
};
// Lays a group of at most kGroup matrices out, chained ones first, longer ones first; the sources are set.
static Plan plan_group(Work* w, int count, int math, int steps, int sms) {
    Plan p;
    long long blocks = 0, wide_tiles[3] = {0, 0, 0};
    double single = 0.0, paired = 0.0;
    for (int k = 0; k < count; ++k) {
        w[k].chained = steps > 1 && chained(w[k].s, math);
        w[k].mb = (w[k].s.m + kBlock - 1) / kBlock;
        w[k].nb = (w[k].s.n + kBlock - 1) / kBlock;
        blocks += w[k].mb * (w[k].mb + 1) / 2;
        // its work in K slices of narrow tiles, one of Q X as 1.5 of them
        const double mk = 2.0 * w[k].mb, nk = 2.0 * w[k].nb, across = 0.375 * nk * mk, pairs = (w[k].mb + 1) / 2;
        single += w[k].mb * (w[k].mb + 1) / 2 * (nk + 2 * mk) + w[k].mb * across;
        paired += 2 * symmetric_count<true>(w[k].mb) * (nk + 2 * mk) + 2 * pairs * across;
        for (int e = 0; e < 3; ++e) wide_tiles[e] += static_cast<long long>(w[k].mb) * (((w[k].s.n + 63) / 64 + (1 << e) - 1) >> e);
    }
    // Where a round has few tiles: two to a block, narrow ones of Q X, and X X^T with its long K in parts, at least eight slices each
    // (together: 1024 x 4096 412 us instead of 491, 1024 x 1024 309 / 385, 512 x 512 203 / 264, 128 x 2048 188 / 303).
    const int fine = 2 * blocks <= sms ? 2 : 1, spare = static_cast<int>(std::max<long long>(1, sms / (blocks * fine)));
    const int wide = wide_tiles[0] <= sms ? 1 : wide_tiles[1] <= sms ? 2 : 4;
    // Pairs of blocks (see the kernel), where every round has tiles for all SMs and little of a pair's work is lost above the diagonal or for an
    // odd row: 4096 x 4096 3.4 ms instead of 4.3, 2048 x 8192 931 us / 1175, eight of 1024 x 4096 1109 / 1256, of 512 x 2048 345 / 390, 30 of 256 x 1024
    // 262 / 284; against it 30 of 640 x 640, five rows each, 814 / 685 (pairs do 1.38 times the work), four of 512 x 2048 among 60 of 128 x 1152
    // 423 / 382.  "f16" gained nothing (4096 x 4096 2.5 ms / 2.35).
    p.pair = math == NML_MATH_3XF16 && fine == 1 && spare == 1 && wide == 4 && sms >= 2 && paired <= 1.2 * single;
    std::sort(w, w + count, [](const Work& a, const Work& b) {
        if (a.chained != b.chained) return a.chained > b.chained;
        if (a.s.m != b.s.m) return a.s.m > b.s.m;
        return a.s.n != b.s.n ? a.s.n > b.s.n : a.s.in < b.s.in;
    });
    int gram = 0, symmetric = 0, update = 0, sum = 0;
    for (int k = 0; k < count; ++k) {
        Work& v = w[k];
        const int c = v.chained ? 0 : 1, own = v.mb * (v.mb + 1) / 2, tiles_of = p.pair ? symmetric_count<true>(v.mb) : own, slices = (v.s.n + 63) / 64;
        if (v.chained) p.first_class = k + 1;
        v.first_sum = p.sums;
        v.sums = static_cast<int>((static_cast<long long>(v.s.m) * v.s.n + kSumElements - 1) / kSumElements);
        p.sums += v.sums;
        v.first_half = p.halves;
        p.halves += v.mb * v.nb * 2;
        v.fine = fine;
        const int most = std::max(1, std::min(spare, slices / 8)), share = (slices + most - 1) / most;
        v.parts = (slices + share - 1) / share;
        v.wide = wide;
        auto tiles = [&](int* first, int* all, int* of_class, int n) {
            *first = *all;
            *all += n;
            *of_class += n;
        };
        tiles(&v.first_gram, &gram, &p.gram_tiles[c], tiles_of * fine * v.parts);
        tiles(&v.first_symmetric, &symmetric, &p.symmetric_tiles[c], tiles_of * fine);
        tiles(&v.first_update, &update, &p.update_tiles[c], (p.pair ? (v.mb + 1) / 2 : v.mb) * ((slices + wide - 1) / wide));
        tiles(&v.first_parts, &sum, &p.sum_tiles[c], v.parts > 1 ? 2 * own : 0);
        for (uint32_t* at : {&v.x[0], &v.x[1]}) *at = p.blocks, p.blocks += v.mb * v.nb;
        v.sym = p.blocks;
        p.blocks += (v.chained ? 7 : 3) * own;
        v.partial = p.blocks;
        if (v.parts > 1) p.blocks += v.parts * own;
    }
    p.identity = p.blocks;
    if (math == NML_MATH_F16) p.blocks += steps;
    p.sums_at = round_up(sizeof(Work) * kGroup, 256);
    p.rounds_at = p.sums_at + round_up(sizeof(double) * p.sums, 256);
    p.done_at = p.rounds_at + round_up(sizeof(Round) * kMaxRounds, 256);
    p.blocks_at = p.done_at + round_up(sizeof(int) * (kGroup + 1), 1024);
    p.blocks_at = round_up(p.blocks_at, 1024);
    p.bytes = p.blocks_at + static_cast<size_t>(p.blocks) * 2 * kPlane;
    return p;
}

// The products of a class, in order; their number.
static int build_ops(const Polynomial& poly, uint32_t identity, bool in_parts, Op* ops) {
    int grown = 0;             // of the present X
    int n = 0, from = 0, gram_before = 0, symmetric_before = 0, wide_before = 0, sum_before = 0;
    auto add = [&](Op op) {
        op.jobs = std::max(op.jobs, 1);
        op.gram_before = gram_before;
        op.symmetric_before = symmetric_before;
        op.wide_before = wide_before;
        op.sum_before = sum_before;
        if (op.kind == SUM) ++sum_before;
        else if (op.kind == ITERATE || op.kind == RESULT) ++wide_before;
        else if (op.kind == POLY && op.gram) ++gram_before;
        else symmetric_before += op.jobs;
        ops[n++] = op;
    };
    // a product of two symmetric matrices stored times 2^el and 2^er, to be stored times 2^eo, + d on the diagonal
    auto symmetric = [](int left, int el, int right, int er, int out, int eo, double d) {
        return Symmetric{left, right, out, static_cast<float>(ldexp(1.0, eo - el - er)), static_cast<float>(ldexp(d, eo))};
    };
    int u = kUpdate, q = kQ;   // the current U and Q
    int eu_last = 0, eq = 0;   // exponents of the last step's U and of Q
    for (int k = 0; k < poly.steps; ++k) {
        const Step& s = poly.step[k];
        Op a = {};             // A and P
        a.kind = POLY;
        a.gram = s.starts;
        a.from = from;
        a.grown = grown;
        if (s.starts) a.job[0] = {0, 0, kGram, static_cast<float>(ldexp(1.0, s.ea)), 0.f};
        else a.job[0] = symmetric(u, eu_last, kT, poly.step[k - 1].et, kGram, s.ea, 0.0);
        a.f1 = static_cast<float>(ldexp(s.c, s.ep - (s.starts ? 0 : eu_last + poly.step[k - 1].et)));
        a.d1 = static_cast<float>(ldexp(s.b, s.ep));
        add(a);
        if (s.starts && in_parts) {
            a.kind = SUM;
            add(a);
        }
        u = s.starts || u != kUpdate ? kUpdate : kUpdate2;
        if (s.starts) q = u, eq = s.eu;
        Op b = {};             // U
        b.kind = PLAIN;
        b.job[0] = symmetric(kPoly, s.ep, kGram, s.ea, u, s.eu, s.a);
        add(b);
        Op c = {};             // T = U A where the chain goes on, and Q = U Q
        c.kind = PLAIN;
        if (!s.ends) c.job[c.jobs++] = symmetric(u, s.eu, kGram, s.ea, kT, s.et, 0.0);
        if (!s.starts) {
            const int to = q == kQ ? kQ2 : kQ;
            c.job[c.jobs++] = symmetric(u, s.eu, q, eq, to, s.eq, 0.0);
            q = to;
            eq = s.eq;
        }
        if (c.jobs) add(c);
        eu_last = s.eu;
        if (s.ends) {
            Op x = {};
            x.kind = k == poly.steps - 1 ? RESULT : ITERATE;
            x.from = from;
            x.left = q;
            x.f1 = static_cast<float>(ldexp(1.0, -eq));
            x.identity = identity + k;
            x.grown = grown | s.grown << kGrownBits;
            grown = s.grown;
            add(x);
            from ^= 1;
        }
    }
    return n;
}

struct Call {
    int in_dtype = NML_F32, out_dtype = NML_F32, math = NML_MATH_3XF16;
    float eps = 0.f;
    Momentum mo = {1.f, 0.f, false, false};
    bool apply = false;
    bool packed = false;  // everything has to be read before anything is written
    float keep = 0.f, rate = 0.f;
    const int* skip = nullptr;
};

template <int N>
static void launch_sums(const Work* w, const Common& c, const Call& call, int blocks, cudaStream_t st) {
    Group<N> g;
    std::copy(w, w + c.count, g.w);
    nml::launch(call.in_dtype == NML_F16 ? ortho_sums_kernel<N, __half> : ortho_sums_kernel<N, float>, blocks, 256, 0, st, g, c, call.mo);
}
// `rounds` of them are set; the others' room does not travel where they are few.
template <int N>
static void launch_pack(const PackParams<kMaxRounds>& all, const Call& call, int blocks, cudaStream_t st) {
    PackParams<N> q = {all.c, all.mo, all.eps, all.halves, all.rounds, all.identity, all.identities, {}, {}};
    std::copy(all.diagonal, all.diagonal + kMaxSteps, q.diagonal);
    std::copy(all.round, all.round + std::min(N, all.rounds), q.round);
    nml::launch(call.in_dtype == NML_F16 ? ortho_pack_kernel<N, __half> : ortho_pack_kernel<N, float>, blocks, 256, 0, st, q);
}
constexpr int kFewRounds = 22;

// Whether a group goes through double precision: see nml_ortho_small.cuh.
static bool all_small(const Work* w, int count) {
    return std::all_of(w, w + count, [](const Work& v) { return v.s.m <= kSmall; });
}
// A chain of steps there amplifies what rounding leaves of a Gram matrix's zero eigenvalues, 2^-53 either way, by kSmallGrowth at most: beyond, negative ones
// come near -1, where the polynomial has no bound (rank 1, 64 x 147, default coefficients: 1e-10 off after 9 steps in one chain, 4e-6 after 12, 0.1 after
// 15, no numbers after 20).  Then X is formed, in fp32, and the next chain starts at its Gram matrix.
constexpr double kSmallGrowth = 1e10;
struct SmallPlan {
    int partials = 0, chunks = 0;
    size_t sums_at = 0, q_at = 0, x_at = 0, bytes = 0;
    size_t x[kGroup];  // where each matrix's X begins behind that
};
static SmallPlan plan_small(Work* w, int count) {
    SmallPlan p;
    for (int k = 0; k < count; ++k) {
        const int chunks = (w[k].s.n + 63) / 64, most = std::min(chunks, kSmallPartials), per = (chunks + most - 1) / most;
        w[k].first_sum = p.partials;
        w[k].sums = (chunks + per - 1) / per;
        p.partials += w[k].sums;
        w[k].first_half = p.chunks;
        p.chunks += chunks;
    }
    p.sums_at = round_up(sizeof(Work) * kGroup, 256);
    p.q_at = p.sums_at + sizeof(double) * kSmall * kSmall * p.partials;
    p.x_at = round_up(p.q_at + sizeof(double) * kSmall * kSmall * count, 256);
    p.bytes = p.x_at;
    for (int k = 0; k < count; ++k) {
        p.x[k] = p.bytes - p.x_at;
        p.bytes += round_up(sizeof(float) * w[k].s.m * w[k].s.n, 256);
    }
    return p;
}
constexpr size_t kSmallStepsSmem = 5 * sizeof(double) * kSmall * kSmallPitch, kSmallResultSmem = 2 * sizeof(double) * kSmall * kSmallPitch;

// The polynomials of the two classes.
struct Steps {
    Polynomial of[kClasses];
};
static bool steps_of(const double* coefficients, int steps, Steps* s) {
    return polynomial(coefficients, steps, true, &s->of[0]) && polynomial(coefficients, steps, false, &s->of[1]);
}

static int run_small(Work* w, int count, const Call& call, const Polynomial& poly, void* workspace, size_t bytes, cudaStream_t st) {
    int* err;
    int sms;
    if (const int rc = nml::current_device(&err, &sms)) return rc;  // (sets the device up)
    const SmallPlan p = plan_small(w, count);
    uint8_t* const base = reinterpret_cast<uint8_t*>(round_up(reinterpret_cast<uintptr_t>(workspace), 1024));
    if (!workspace || base + p.bytes > static_cast<uint8_t*>(workspace) + bytes) return NML_ERR_WORKSPACE;
    const Common c = {reinterpret_cast<Work*>(base), reinterpret_cast<double*>(base + p.sums_at), nullptr, nullptr, nullptr, call.skip, count};
    double* const q = reinterpret_cast<double*>(base + p.q_at);
    // Three launches a chain.  Where everything has to be read before a result is written, the last chain has no steps, and takes X to its place.
    for (int first = 0, chains = 0; first < poly.steps || call.packed; ++chains) {
        const bool starts = chains == 0;
        int end = first;
        for (double growth = 1.0; end < poly.steps && (end == first || growth * poly.step[end].amplified <= kSmallGrowth); ++end) growth *= poly.step[end].amplified;
        const bool last = end == poly.steps && (!call.packed || first == end);
        const bool half = starts && call.in_dtype == NML_F16;
        const Momentum mo = starts ? call.mo : Call().mo;
        auto gram = [&](auto n) {
            constexpr int N = decltype(n)::value;
            Group<N> g;
            std::copy(w, w + count, g.w);
            for (int k = 0; k < count; ++k) {
                Source& s = g.w[k].s;
                float* const x = reinterpret_cast<float*>(base + p.x_at + p.x[k]);
                if (!starts) s.in = x, s.in_i = s.n, s.in_j = 1;
                if (!last) s.out = x, s.out_i = s.n, s.out_j = 1;
            }
            nml::launch(half ? small_gram_kernel<N, __half> : small_gram_kernel<N, float>, p.partials, 256, 0, st, g, c, mo);
        };
        if (count <= 8) gram(std::integral_constant<int, 8>());
        else gram(std::integral_constant<int, kGroup>());
        SmallSteps s = {c, q, call.eps, starts, end - first, {}, {}, {}};
        for (int k = first; k < end; ++k) s.a[k - first] = poly.step[k].a, s.b[k - first] = poly.step[k].b, s.k[k - first] = poly.step[k].c;
        nml::launch(small_steps_kernel, count, 32 * kStepsWarps, kSmallStepsSmem, st, s);
        const SmallResult r = {c, q, mo, last && call.out_dtype == NML_F16, last && call.apply, call.keep, call.rate};
        nml::launch(half ? small_result_kernel<__half> : small_result_kernel<float>, p.chunks, 256, kSmallResultSmem, st, r);
        NMLO_CUDA(cudaGetLastError());
        nml::count_launches(3);
        if (last) break;
        first = end;
    }
    return NML_OK;
}

// One group: three launches (a chain).
static int run_group(Work* w, int count, const Call& call, const Steps& steps, void* workspace, size_t bytes, cudaStream_t st) {
    if (all_small(w, count)) return run_small(w, count, call, steps.of[1], workspace, bytes, st);
    int* err;
    int sms;
    if (const int rc = nml::current_device(&err, &sms)) return rc;
    const Plan p = plan_group(w, count, call.math, steps.of[0].steps, sms);
    uint8_t* const base = reinterpret_cast<uint8_t*>(round_up(reinterpret_cast<uintptr_t>(workspace), 1024));
    if (!workspace || base + p.bytes > static_cast<uint8_t*>(workspace) + bytes) return NML_ERR_WORKSPACE;
    for (int k = 0; k < count; ++k) {
        const double elements = static_cast<double>(w[k].s.m) * w[k].s.n;
        const int e = std::min(exponent_below(steps.of[w[k].chained ? 0 : 1].largest), static_cast<int>(lround(0.5 * log2(elements))));
        w[k].sx = e;
    }
    const Common c = {reinterpret_cast<Work*>(base), reinterpret_cast<double*>(base + p.sums_at), reinterpret_cast<Round*>(base + p.rounds_at),
                      reinterpret_cast<int*>(base + p.done_at), base + p.blocks_at, call.skip, count};

    // rounds: a product of each class, with as many tiles as its matrices have
    PackParams<kMaxRounds> pack = {c, call.mo, call.eps, p.halves, 0, p.identity, call.math == NML_MATH_F16 ? steps.of[1].steps : 0, {}, {}};
    Op ops[kClasses][kMaxRounds];
    int number[kClasses];
    for (int cls = 0; cls < kClasses; ++cls) number[cls] = build_ops(steps.of[cls], p.identity, p.sum_tiles[cls] > 0, ops[cls]);
    if (p.first_class == 0) number[0] = 0;
    if (p.first_class == count) number[1] = 0;
    pack.rounds = std::max(number[0], number[1]);
    long long tiles = 0, widest = 0;
    for (int r = 0; r < pack.rounds; ++r) {
        Round& round = pack.round[r];
        round.first = static_cast<int>(tiles);
        round.of_first = 0;
        for (int cls = 0; cls < kClasses; ++cls) {
            if (r >= number[cls]) continue;
            const Op& op = round.op[cls] = ops[cls][r];
            const long long n = op.kind == ITERATE || op.kind == RESULT ? p.update_tiles[cls]
                                : op.kind == SUM ? p.sum_tiles[cls] : op.kind == POLY && op.gram ? p.gram_tiles[cls]
                                : static_cast<long long>(op.jobs) * p.symmetric_tiles[cls];
            if (cls == 0) round.of_first = static_cast<int>(n);
            tiles += n;
        }
        widest = std::max(widest, tiles - round.first);
    }
    if (tiles > (1 << 27)) return NML_ERR_UNSUPPORTED;
    // no wait is longer than all the work by one block, at 2 us a K slice (0.8 measured)
    double slices = 0.0;
    for (int k = 0; k < count; ++k) {
        const double m = w[k].s.m / 64 + 1, n = w[k].s.n / 64 + 1, t = w[k].mb * (w[k].mb + 1) / 2;
        slices += steps.of[1].steps * 2 * (t * n + 3 * t * m + w[k].mb * n * (m + 2));
    }

    if (count <= 8) launch_sums<8>(w, c, call, p.sums, st);
    else launch_sums<kGroup>(w, c, call, p.sums, st);
    for (int k = 0; k < steps.of[1].steps; ++k) pack.diagonal[k] = static_cast<float>(ldexp(steps.of[1].step[k].a, steps.of[1].step[k].eu));
    const int blocks = p.halves + 2 * pack.identities + 1;
    if (pack.rounds <= kFewRounds) launch_pack<kFewRounds>(pack, call, blocks, st);
    else launch_pack<kMaxRounds>(pack, call, blocks, st);
    ProductParams q = {{}, c, err, static_cast<unsigned long long>(1.5e9 + 2e3 * slices), pack.rounds, static_cast<int>(tiles), p.first_class,
                             call.out_dtype == NML_F16, call.apply, call.keep, call.rate};
    if (p.pair)
        for (int e = 0; e < kMaps; ++e) {
            const uint64_t dims[5] = {256, 16, 2, 2, 2ull * p.blocks};
            const uint32_t box[5] = {256, 16, e == MAP_HALF ? 2u : 1u, e == MAP_ACROSS ? 2u : 1u, 2};
            if (const int rc = nml::encode_box(&q.map[e], c.blocks, 5, dims, box)) return rc;
        }
    // (no more blocks than a round has tiles)
    const int each = p.pair ? 2 : 1, grid = each * static_cast<int>(std::min<long long>(widest, sms / each));
    nml::launch_with(nml::overlaps(grid, nml::kSms), each,
                     call.math == NML_MATH_F16 ? ortho_product_kernel<1, false> : p.pair ? ortho_product_kernel<2, true> : ortho_product_kernel<2, false>,
                     grid, kThreads, kProductSmem, st, q);
    NMLO_CUDA(cudaGetLastError());
    nml::count_launches(3);
    return NML_OK;
}

static bool math_ok(int math) { return math == NML_MATH_F16 || math == NML_MATH_3XF16; }
constexpr int kLongest = 1 << 24;  // (indexes of blocks, tiles and sums are 32-bit)
static bool size_ok(int rows, int cols) {
    return rows > 0 && cols > 0 && rows <= kLongest && cols <= kLongest && static_cast<long long>(rows) * cols <= (1ll << 36);
}
static void set_sizes(Source& s, int rows, int cols) {
    s.m = std::min(rows, cols);
    s.n = std::max(rows, cols);
}
static bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Whether what a step writes is in one place each: a parameter that is listed twice would be updated by two blocks at a time.  Gradients may be shared,
// but lie apart from all that.
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
        for (int k = 0; k < count; ++k) {
            const uintptr_t from = reinterpret_cast<uintptr_t>(params[k].grad);
            const uintptr_t to = from + 4 * static_cast<uintptr_t>(std::max(params[k].rows, 1)) * params[k].cols;
            const auto next = std::lower_bound(r.begin(), r.end(), Range(to, 0));  // the first one that begins at its end or behind
            if (next != r.begin() && std::prev(next)->second > from) return false;
        }
        return true;
    } catch (...) {
        return false;
    }
}
// The memory of a matrix (one of its strides is 1).
static nml::Runs runs_of(const void* p, int rows, int cols, long long row, long long col, long long size) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (col == 1 && (row >= cols || rows == 1)) return {at, rows, cols * size, row * size};
    return {at, cols, rows * size, col * size};
}
enum Places { APART, OVER_INPUTS, CLASH };
// Where results lie: apart from one another, and each apart from its own matrix or where that one does (CLASH otherwise); OVER_INPUTS: some lie over other
// matrices that are read.
static Places places(const nml_matrix* matrices, int count, long long in_size, long long out_size) {
    auto in = [&](int k) { return runs_of(matrices[k].in, matrices[k].rows, matrices[k].cols, matrices[k].in_row, matrices[k].in_col, in_size); };
    auto out = [&](int k) { return runs_of(matrices[k].out, matrices[k].rows, matrices[k].cols, matrices[k].out_row, matrices[k].out_col, out_size); };
    for (int k = 0; k < count; ++k)
        if (matrices[k].in != matrices[k].out && overlap(in(k), out(k))) return CLASH;
    if (count < 2) return APART;
    struct Piece {
        nml::Runs runs;
        int k;
    };
    try {
        std::vector<Piece> ins, outs;
        std::vector<uintptr_t> reach;  // the furthest end of the first ones of `ins`
        ins.reserve(count), outs.reserve(count), reach.reserve(count);
        for (int k = 0; k < count; ++k) ins.push_back({in(k), k}), outs.push_back({out(k), k});
        auto by_place = [](const Piece& a, const Piece& b) { return a.runs.at < b.runs.at; };
        std::sort(ins.begin(), ins.end(), by_place);
        std::sort(outs.begin(), outs.end(), by_place);
        for (const Piece& p : ins) reach.push_back(std::max(p.runs.end(), reach.empty() ? 0 : reach.back()));
        Places found = APART;
        for (int o = 0; o < count; ++o) {
            const Piece& p = outs[o];
            for (int e = o + 1; e < count && outs[e].runs.at < p.runs.end(); ++e)
                if (overlap(p.runs, outs[e].runs)) return CLASH;
            if (found == OVER_INPUTS) continue;
            for (size_t e = std::upper_bound(reach.begin(), reach.end(), p.runs.at) - reach.begin(); e < ins.size() && ins[e].runs.at < p.runs.end(); ++e)
                if (ins[e].k != p.k && overlap(p.runs, ins[e].runs)) {
                    found = OVER_INPUTS;
                    break;
                }
        }
        return found;
    } catch (...) {
        return CLASH;
    }
}

// Workspace of the largest group of `count` matrices whose sizes `size(k, source)` sets (false: not a matrix, left out).
template <class F>
static int workspace_of(int count, int math, int steps, F&& size, size_t* bytes) {
    Work w[kGroup];
    *bytes = 0;
    int sms = nml::usable_sms(), filled = 0;
    for (int k = 0; k <= count; ++k) {
        if (filled == kGroup || (k == count && filled > 0)) {
            *bytes = std::max(*bytes, (all_small(w, filled) ? plan_small(w, filled).bytes : plan_group(w, filled, math, steps, sms).bytes) + 1024);
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

// Whether the product kernels have the registers that their split among the warps counts on; a build that gave them others would wait for registers
// for good, so such a build refuses the calls of this file, and no others.  (Of the build, hence the same on every device.)
static std::atomic<bool> g_split_holds{false};
// Sets the device up.
static int products_run() {
    int* err;
    int sms;
    if (const int rc = nml::current_device(&err, &sms)) return rc;
    return g_split_holds.load(std::memory_order_relaxed) ? NML_OK : NML_ERR_UNSUPPORTED;
}

int nml::prepare_ortho_kernels() {
    cudaFuncAttributes a;
    bool holds = true;
    for (auto f : {ortho_product_kernel<1, false>, ortho_product_kernel<2, false>, ortho_product_kernel<2, true>}) {
        NMLO_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kProductSmem)));
        NMLO_CUDA(cudaFuncGetAttributes(&a, f));
        holds = holds && a.numRegs == kLaunchRegs;
    }
    g_split_holds.store(holds, std::memory_order_relaxed);
    NMLO_CUDA(cudaFuncSetAttribute(small_steps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmallStepsSmem)));
    NMLO_CUDA(cudaFuncSetAttribute(small_result_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmallResultSmem)));
    NMLO_CUDA(cudaFuncSetAttribute(small_result_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmallResultSmem)));
    const void* others[] = {(const void*)small_gram_kernel<8, float>, (const void*)small_gram_kernel<8, __half>,
                            (const void*)small_gram_kernel<kGroup, float>, (const void*)small_gram_kernel<kGroup, __half>, (const void*)ortho_sums_kernel<8, float>, (const void*)ortho_sums_kernel<8, __half>,
                            (const void*)ortho_sums_kernel<kGroup, float>, (const void*)ortho_sums_kernel<kGroup, __half>,
                            (const void*)ortho_pack_kernel<kFewRounds, float>, (const void*)ortho_pack_kernel<kFewRounds, __half>,
                            (const void*)ortho_pack_kernel<kMaxRounds, float>, (const void*)ortho_pack_kernel<kMaxRounds, __half>,
                            (const void*)momentum_vectors_kernel};
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

int nml_orthogonalize(const nml_matrix* matrices, int count, int in_dtype, int out_dtype, int math, int steps, const double* coefficients,
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
        // in place: element by element
        if (x.in == x.out && (in_dtype != out_dtype || x.in_row != x.out_row || x.in_col != x.out_col)) return NML_ERR_INVALID;
    }
    // Tiles are packed from all matrices of a group before the first result is written, and small matrices' X can be formed elsewhere first; but from one group
    // to the next, results are written while others' matrices are still to be read.
    const Places where = places(matrices, count, in_dtype == NML_F16 ? 2 : 4, out_dtype == NML_F16 ? 2 : 4);
    if (where == CLASH || (where == OVER_INPUTS && count > kGroup)) return NML_ERR_INVALID;
    Steps poly;
    if (!steps_of(coefficients, steps, &poly)) return NML_ERR_UNSUPPORTED;
    if (count > 0 && (!workspace || workspace_bytes < need)) return NML_ERR_WORKSPACE;
    if (count > 0)
        if (const int rc = products_run()) return rc;
    Call call;
    call.in_dtype = in_dtype;
    call.out_dtype = out_dtype;
    call.math = math;
    call.eps = eps;
    call.packed = where == OVER_INPUTS;
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

int nml_muon_step(const nml_muon_param* params, int count, int math, int steps, const double* coefficients, float eps, float lr, float momentum,
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
    Steps poly;
    if (!steps_of(coefficients, steps, &poly)) return NML_ERR_UNSUPPORTED;
    if (need > 0 && (!workspace || workspace_bytes < need)) return NML_ERR_WORKSPACE;
    if (need > 0)
        if (const int rc = products_run()) return rc;  // (before anything is updated)
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
    auto run_vectors = [&]() -> int {
        int* err;
        int sms;
        if (const int rc = nml::current_device(&err, &sms)) return rc;
        nml::launch(momentum_vectors_kernel, others, 256, 0, st, vectors);
        NMLO_CUDA(cudaGetLastError());
        nml::count_launches(1);
        others = 0;
        return NML_OK;
    };
    for (int k = 0; k <= count; ++k) {
        if (matrices == kGroup || (k == count && matrices > 0)) {
            if (const int rc = run_group(w, matrices, call, poly, workspace, workspace_bytes, st)) return rc;
            matrices = 0;
        }
        if (k == count) break;
        const nml_muon_param& p = params[k];
        if (p.rows == 0) {
            for (long long from = 0; from < p.cols; from += kVectorPiece) {
                __half* const half = static_cast<__half*>(p.param_f16);
                vectors.v[others++] = {p.param + from, p.grad + from, p.momentum + from, half ? half + from : nullptr,
                                       static_cast<int>(std::min<long long>(kVectorPiece, p.cols - from))};
                if (others == kVectors)
                    if (const int rc = run_vectors()) return rc;
            }
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
    return others > 0 ? run_vectors() : NML_OK;
}

}  // extern "C"
