// Orthogonalised matrices whose short side is at most 64: everything about the long side in two passes over the matrix, and the steps
// on m x m matrices between them.
//
//   A = G G^T / (|G| + eps)^2;  U_k = a I + b A + c A^2,  A <- U_k A U_k,  Q <- U_k Q;  result = Q G / (|G| + eps)
//
// (all of them polynomials of the first A, so symmetric; |G|^2 is the trace of G G^T).  The steps square the condition number and
// amplify the error of A by up to max u^2 each (a^2 = 11.9 with the default coefficients), so this is done in double, and in one chain only as far as
// its steps together amplify it by 1e10: five default steps do by 2.3e5, 2^-53 of which is 3e-11, nine by 5e9; and the result is rounded once.
// With tiles of 128 in three products of halves a matrix of 64 x 147 took 116 us, 15 products of one tile, 7 us each: loads, flags and
// stores.  Here it takes 59 us in three launches: partial Gram matrices of 64 columns a block; the steps, a block to a matrix; Q G, 64 columns a block
// (8, 52 and 11 us where each is timed alone, launch included).
// The steps are bound by one block's double-precision pipe and by the barriers between its products: 64 FMAs a clock and SM, from registers or by mma.sync
// alike (both measured), so the lower blocks of a product of 64 x 64 matrices take 2304 clocks and the 17 of five steps 39 thousand; the launch takes 99
// thousand, of which the pipe is busy for 53 % (with what is done to the elements).  mma.sync needs a quarter of the shared-memory reads.
#pragma once

namespace nml_ortho {

constexpr int kSmall = 64;             // short side, at most
constexpr int kSmallPartials = 24;     // of a matrix: blocks of the first launch
constexpr int kSmallPitch = 68;        // doubles: four rows of an 8 x 4 fragment meet every bank

// Sixty-four columns of a matrix as doubles in shared memory, [row][column] or (across) [column][row]; zeros beyond the edges.
template <typename T, bool kAcross>
__device__ __forceinline__ void load_columns(const Source& s, const Momentum& mo, int j0, bool advance, double (*x)[kSmallPitch]) {
    const bool turned = s.in_i == 1 && s.in_j != 1;  // memory runs along i
    const int along = threadIdx.x & 63, other = threadIdx.x >> 6;
    const T* const in = static_cast<const T*>(s.in);
#pragma unroll 1
    for (int e0 = 0; e0 < 16; e0 += 8) {
        float v[8], b[8];
        long long at[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int o = other + 4 * (e0 + e), i = turned ? along : o, j = j0 + (turned ? o : along);
            at[e] = i < s.m && j < s.n ? i * s.in_i + j * s.in_j : -1;
            v[e] = at[e] >= 0 ? load_as_float(in + at[e]) : 0.f;
            b[e] = mo.on && at[e] >= 0 ? load_global(s.momentum + at[e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int o = other + 4 * (e0 + e), i = turned ? along : o, j = turned ? o : along;
            if (mo.on) {
                const float g = v[e] * mo.inv_scale;
                if (advance) {
                    b[e] = mo.momentum * b[e] + g;  // the new momentum
                    if (at[e] >= 0) s.momentum[at[e]] = b[e];
                }
                v[e] = mo.nesterov ? g + mo.momentum * b[e] : b[e];
            }
            x[kAcross ? j : i][kAcross ? i : j] = static_cast<double>(v[e]);
        }
    }
}

// d += l r^T: 8 x 8 elements of the products of 8 rows of each along k, by a warp.  A lane holds row lane / 4, columns 2 (lane % 4) and the next.
__device__ __forceinline__ void multiply8(const double (*l)[kSmallPitch], const double (*r)[kSmallPitch], int k, double (&d)[2]) {
    const int lane = threadIdx.x & 31;
    const double a = l[lane >> 2][k + (lane & 3)], b = r[lane >> 2][k + (lane & 3)];
    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}
// The lower 8 x 8 tiles of l r^T, t = warp, warp + kWarps, ... to a warp; kTiles x kWarps are at least 36.
template <int kWarps, int kTiles>
__device__ __forceinline__ void multiply_lower(const double (*l)[kSmallPitch], const double (*r)[kSmallPitch], int tiles, int depth, double (&d)[kTiles][2]) {
    const int warp = threadIdx.x >> 5;
    int row[kTiles], column[kTiles];
#pragma unroll
    for (int e = 0; e < kTiles; ++e) {
        const int t = warp + kWarps * e;
        row[e] = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
        column[e] = t - row[e] * (row[e] + 1) / 2;
    }
#pragma unroll 2
    for (int k = 0; k < depth; k += 4)
#pragma unroll
        for (int e = 0; e < kTiles; ++e)
            if (warp + kWarps * e < tiles) multiply8(l + 8 * row[e], r + 8 * column[e], k, d[e]);
}
// f(value, i, j) for this lane's elements of them.
template <int kWarps, int kTiles, class F>
__device__ __forceinline__ void each_lower(int tiles, const double (&d)[kTiles][2], F&& f) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < kTiles; ++e) {
        const int t = warp + kWarps * e;
        if (t >= tiles) continue;
        const int row = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f), column = t - row * (row + 1) / 2;
        const int i = 8 * row + (lane >> 2), j = 8 * column + 2 * (lane & 3);
        f(d[e][0], i, j);
        f(d[e][1], i, j + 1);
    }
}
__device__ __forceinline__ int small_side(int m) { return (m + 7) & ~7; }
__device__ __forceinline__ int small_lower(int side) { return side / 8 * (side / 8 + 1) / 2; }

// Partial Gram matrices: a block to `per` times 64 columns of a matrix.  The first block leaves the group's table in the workspace.
template <int N, typename T>
__global__ void __launch_bounds__(256) small_gram_kernel(const __grid_constant__ Group<N> group, const Common c, const Momentum mo) {
    pdl_enter();
    __shared__ double x[kSmall][kSmallPitch];
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < c.count; i += blockDim.x) c.table[i] = group.w[i];
    if (skipped(c.skip)) return;
    int lo = 0, hi = c.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (group.w[mid].first_sum <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
    }
    const Work& w = group.w[lo];
    const int part = blockIdx.x - w.first_sum, tiles = small_lower(small_side(w.s.m)), chunks = (w.s.n + 63) / 64, per = (chunks + w.sums - 1) / w.sums;
    double d[5][2] = {};
    for (int e = part * per; e < min(chunks, (part + 1) * per); ++e) {
        __syncthreads();
        load_columns<T, false>(w.s, mo, e * 64, true, x);
        __syncthreads();
        multiply_lower<8>(x, x, tiles, min(64, (w.s.n - e * 64 + 3) & ~3), d);
    }
    double* const out = c.sums + static_cast<size_t>(blockIdx.x) * kSmall * kSmall;
    each_lower<8>(tiles, d, [&](double v, int i, int j) { out[i * kSmall + j] = v; });
}

struct SmallSteps {
    Common c;
    double* q;       // results, kSmall x kSmall to a matrix
    double eps;
    bool starts;     // at G, which is normalised
    int steps;       // none: Q is 1
    double a[kMaxSteps], b[kMaxSteps], k[kMaxSteps];  // coefficients
};
// The steps, a block to a matrix.
constexpr int kStepsWarps = 16;
__global__ void __launch_bounds__(32 * kStepsWarps) small_steps_kernel(const __grid_constant__ SmallSteps P) {
    pdl_enter();
    if (skipped(P.c.skip)) return;
    extern __shared__ double room[];
    typedef double (*Matrix)[kSmallPitch];
    constexpr int kOne = kSmall * kSmallPitch;
    __shared__ double inverse;
    Matrix A = reinterpret_cast<Matrix>(room), U = reinterpret_cast<Matrix>(room + kOne), T = reinterpret_cast<Matrix>(room + 2 * kOne),
           Q = reinterpret_cast<Matrix>(room + 3 * kOne), next = reinterpret_cast<Matrix>(room + 4 * kOne);
    const Work w = load_work(P.c.table + blockIdx.x);
    const int m = small_side(w.s.m), tiles = small_lower(m), tid = threadIdx.x, i0 = tid >> 6, j0 = tid & 63;
    auto each = [&](auto&& f) {  // all elements
        if (j0 < m)
            for (int i = i0; i < m; i += kStepsWarps / 2) f(i, j0);
    };
    // the sum of the partial ones, in a fixed order; the lower blocks, mirrored
#pragma unroll 2
    for (int i = i0; i < m; i += kStepsWarps / 2) {
        if (j0 > i) continue;
        const double* from = P.c.sums + static_cast<size_t>(w.first_sum) * kSmall * kSmall + i * kSmall + j0;
        double s = 0.0;
#pragma unroll 8
        for (int p = 0; p < w.sums; ++p) s += load_double(from + static_cast<size_t>(p) * kSmall * kSmall);
        A[i][j0] = A[j0][i] = s;
    }
    __syncthreads();
    if (tid < 32) {
        double trace = (tid < m ? A[tid][tid] : 0.0) + (tid + 32 < m ? A[tid + 32][tid + 32] : 0.0);
#pragma unroll
        for (int o = 16; o > 0; o /= 2) trace += __shfl_xor_sync(0xffffffffu, trace, o);
        const double norm = sqrt(trace) + P.eps;
        if (tid == 0) inverse = !P.starts ? 1.0 : norm == 0.0 ? 0.0 : 1.0 / norm;  // (zeros stay zeros without an eps too)
    }
    __syncthreads();
    const double inv = inverse;
    each([&](int i, int j) { A[i][j] *= inv * inv; });
    __syncthreads();
    // out = f(l r, i, j) of two symmetric matrices, both triangles
    auto product = [&](Matrix l, Matrix r, Matrix out, auto&& f) {
        double d[3][2] = {};
        multiply_lower<kStepsWarps>(l, r, tiles, m, d);
        each_lower<kStepsWarps>(tiles, d, [&](double v, int i, int j) {
            if (i >= j) out[i][j] = out[j][i] = f(v, i, j);
        });
    };
    const auto plain = [](double d, int, int) { return d; };
    if (P.steps == 0) each([&](int i, int j) { Q[i][j] = i == j ? 1.0 : 0.0; });
    for (int k = 0; k < P.steps; ++k) {
        const bool last = k + 1 == P.steps;
        product(A, A, U, [&](double d, int i, int j) { return P.k[k] * d + P.b[k] * A[i][j] + (i == j ? P.a[k] : 0.0); });
        __syncthreads();
        if (k == 0) {
            each([&](int i, int j) { Q[i][j] = U[i][j]; });
        } else {
            product(U, Q, next, plain);
            Matrix t = Q;
            Q = next;
            next = t;
        }
        if (!last) {
            product(U, A, T, plain);
            __syncthreads();
            product(U, T, A, plain);
        }
        __syncthreads();
    }
    each([&](int i, int j) { P.q[static_cast<size_t>(blockIdx.x) * kSmall * kSmall + i * kSmall + j] = Q[i][j] * inv; });
}

// Q G: a block to 64 columns of a matrix.
struct SmallResult {
    Common c;
    const double* q;
    Momentum mo;
    int out_half;
    bool apply;
    float keep, rate;
};
template <typename T>
__global__ void __launch_bounds__(256) small_result_kernel(const __grid_constant__ SmallResult P) {
    pdl_enter();
    if (skipped(P.c.skip)) return;
    extern __shared__ double room[];
    typedef double (*Matrix)[kSmallPitch];
    Matrix x = reinterpret_cast<Matrix>(room), q = reinterpret_cast<Matrix>(room + kSmall * kSmallPitch);
    __shared__ int first[kGroup];
    const int tid = threadIdx.x;
    for (int i = tid; i < P.c.count; i += 256) first[i] = load_global(&P.c.table[i].first_half);
    __syncthreads();
    const int k = owner_of(first, P.c.count, blockIdx.x);
    const Work w = load_work(P.c.table + k);
    const Source& s = w.s;
    const int j0 = (blockIdx.x - first[k]) * 64, m = small_side(s.m), warp = tid >> 5, lane = tid & 31;
    load_columns<T, true>(s, P.mo, j0, false, x);
    if ((tid & 63) < m)
#pragma unroll 4
        for (int i = tid >> 6; i < m; i += 4) q[i][tid & 63] = load_double(P.q + static_cast<size_t>(k) * kSmall * kSmall + i * kSmall + (tid & 63));
    __syncthreads();
    // eight columns to a warp
    double d[kSmall / 8][2] = {};
#pragma unroll 2
    for (int e = 0; e < m; e += 4)
#pragma unroll
        for (int p = 0; p < kSmall / 8; ++p)
            if (8 * p < m) multiply8(q + 8 * p, x + 8 * warp, e, d[p]);
    __syncthreads();
    // through shared memory, so that the lanes of a warp lie densely in the result, along its columns or (turned) its rows
#pragma unroll
    for (int p = 0; p < kSmall / 8; ++p)
        if (8 * p < m) {
            q[8 * p + (lane >> 2)][8 * warp + 2 * (lane & 3)] = d[p][0];
            q[8 * p + (lane >> 2)][8 * warp + 2 * (lane & 3) + 1] = d[p][1];
        }
    __syncthreads();
    const bool turned = s.out_i == 1 && s.out_j != 1;
    ProductParams out = {};
    out.out_half = P.out_half;
    out.apply = P.apply;
    out.keep = P.keep;
    const float rate = P.rate * s.scale;
#pragma unroll 4
    for (int e = tid >> 6; e < 64; e += 4) {
        const int i = turned ? tid & 63 : e, j = turned ? e : tid & 63;
        if (i < s.m && j0 + j < s.n)
            put1(out, static_cast<uint8_t*>(s.out), reinterpret_cast<uint8_t*>(s.half), i * s.out_i + (j0 + j) * s.out_j, static_cast<float>(q[i][j]), rate);
    }
}

}  // namespace nml_ortho
