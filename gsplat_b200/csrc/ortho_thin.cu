// Newton-Schulz orthogonalisation of many thin matrices (short side S <= 4, long
// side L <= 128): forward, backward and the whole Muon step, one launch each.
//
// A group of 2^g lanes holds one matrix in registers, kRows rows of S values a
// lane, and every step stays there: the S x S Gram matrix is summed over the group with
// shuffles, its polynomial is a handful of FMAs that every lane repeats, and
// X (a I + B) is one S x S product a row. The arithmetic is 32-bit throughout.
// Memory is read and written once, which bounds the large batches; rows past L
// are zeros, which the iteration leaves zero.
#include "ortho.cuh"

namespace gsb {

constexpr int kThinRows = 4;
constexpr int kThinThreads = 128;
constexpr int kThinMaxShort = 4;
constexpr int kThinMaxLong = kThinRows * 32;

bool ortho_is_thin(int rows, int cols) {
    const int s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    return s <= kThinMaxShort && l <= kThinMaxLong;
}

template <int S> struct Sym { // symmetric S x S, upper triangle by rows
    float v[S * (S + 1) / 2];
    __device__ __forceinline__ static constexpr int at(int i, int j) {
        return i <= j ? i * S - i * (i - 1) / 2 + (j - i) : at(j, i);
    }
    __device__ __forceinline__ float operator()(int i, int j) const { return v[at(i, j)]; }
    __device__ __forceinline__ float &operator()(int i, int j) { return v[at(i, j)]; }
};

template <typename T> __device__ __forceinline__ T group_sum(T v, int group) {
    for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// sum over the group of X^T Y + Y^T X (twice the Gram matrix for X = Y), halved
// for X = Y.
template <int S>
__device__ __forceinline__ Sym<S> gram(const float x[kThinRows][S], int group) {
    Sym<S> a;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = i; j < S; ++j) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < kThinRows; ++r) s = fmaf(x[r][i], x[r][j], s);
            a(i, j) = group_sum(s, group);
        }
    return a;
}
template <int S>
__device__ __forceinline__ Sym<S> cross(const float x[kThinRows][S], const float y[kThinRows][S], int group) {
    Sym<S> a;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = i; j < S; ++j) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < kThinRows; ++r) s = fmaf(x[r][i], y[r][j], fmaf(y[r][i], x[r][j], s));
            a(i, j) = group_sum(s, group);
        }
    return a;
}

// b A + c A A
template <int S> __device__ __forceinline__ Sym<S> poly(const Sym<S> &a, float b, float c) {
    Sym<S> r;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = i; j < S; ++j) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < S; ++k) s = fmaf(a(i, k), a(k, j), s);
            r(i, j) = fmaf(b, a(i, j), c * s);
        }
    return r;
}

// X <- a X + X B
template <int S> __device__ __forceinline__ void apply(float x[kThinRows][S], const Sym<S> &B, float a) {
#pragma unroll
    for (int r = 0; r < kThinRows; ++r) {
        float t[S];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            t[j] = a * x[r][j];
#pragma unroll
            for (int k = 0; k < S; ++k) t[j] = fmaf(x[r][k], B(k, j), t[j]);
        }
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = t[j];
    }
}

// The Frobenius norm over the group, summed in 64 bits (any finite input).
template <int S> __device__ __forceinline__ float frobenius(const float x[kThinRows][S], int group) {
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) s = fma((double)x[r][j], (double)x[r][j], s);
    return (float)sqrt(group_sum(s, group));
}

struct ThinShape {
    long long batch;
    int L, S, group;
    long long row_step, col_step; // element (l, s) of a matrix at l * row_step + s * col_step
};

template <int S>
__device__ __forceinline__ void thin_iterate(float x[kThinRows][S], const OrthoCoefficients &co, int group) {
    for (int k = 0; k < co.steps; ++k)
        apply<S>(x, poly<S>(gram<S>(x, group), co.c[k][1], co.c[k][2]), co.c[k][0]);
}

template <typename T, int S>
__global__ void __launch_bounds__(kThinThreads)
    thin_fwd_kernel(ThinShape sh, const T *__restrict__ x_in, T *__restrict__ y, const OrthoCoefficients co, float eps) {
    const int lane = threadIdx.x & (sh.group - 1);
    const long long b = ((long long)blockIdx.x * kThinThreads + threadIdx.x) / sh.group;
    const bool live = b < sh.batch; // the whole group alike; idle groups still shuffle
    const size_t base = (size_t)b * sh.L * S;
    float x[kThinRows][S];
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            x[r][j] = live && l < sh.L ? to_f32(x_in[base + l * sh.row_step + j * sh.col_step]) : 0.f;
        }
    const float norm = frobenius<S>(x, sh.group);
    const float d = norm < eps ? eps : norm;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] / d;
    thin_iterate<S>(x, co, sh.group);
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            if (live && l < sh.L) y[base + l * sh.row_step + j * sh.col_step] = from_f32<T>(x[r][j]);
        }
}

// The backward keeps every step's X in shared memory, [step][value][thread].
template <typename T, int S>
__global__ void __launch_bounds__(kThinThreads)
    thin_bwd_kernel(ThinShape sh, const T *__restrict__ x_in, const T *__restrict__ v_y, T *__restrict__ v_x,
                    const OrthoCoefficients co, float eps) {
    extern __shared__ float kept[];
    const int lane = threadIdx.x & (sh.group - 1);
    const long long b = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / sh.group;
    const bool live = b < sh.batch;
    const size_t base = (size_t)b * sh.L * S;
    float x[kThinRows][S], g[kThinRows][S];
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            const bool in = live && l < sh.L;
            const size_t at = base + l * sh.row_step + j * sh.col_step;
            x[r][j] = in ? to_f32(x_in[at]) : 0.f;
            g[r][j] = in ? to_f32(v_y[at]) : 0.f;
        }
    const float norm = frobenius<S>(x, sh.group);
    const float d = norm < eps ? eps : norm;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] / d;
    for (int k = 0; k < co.steps; ++k) {
#pragma unroll
        for (int r = 0; r < kThinRows; ++r)
#pragma unroll
            for (int j = 0; j < S; ++j)
                kept[((k * kThinRows + r) * S + j) * blockDim.x + threadIdx.x] = x[r][j];
        if (k + 1 < co.steps)
            apply<S>(x, poly<S>(gram<S>(x, sh.group), co.c[k][1], co.c[k][2]), co.c[k][0]);
    }
    for (int k = co.steps - 1; k >= 0; --k) {
        const float ca = co.c[k][0], cb = co.c[k][1], cc = co.c[k][2];
#pragma unroll
        for (int r = 0; r < kThinRows; ++r)
#pragma unroll
            for (int j = 0; j < S; ++j)
                x[r][j] = kept[((k * kThinRows + r) * S + j) * blockDim.x + threadIdx.x];
        const Sym<S> A = gram<S>(x, sh.group), B = poly<S>(A, cb, cc), Q = cross<S>(x, g, sh.group);
        Sym<S> t; // b Q + c (Q A + A Q)
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = i; j < S; ++j) {
                float s = 0.f;
#pragma unroll
                for (int m = 0; m < S; ++m) s = fmaf(Q(i, m), A(m, j), fmaf(A(i, m), Q(m, j), s));
                t(i, j) = fmaf(cb, Q(i, j), cc * s);
            }
        apply<S>(g, B, ca); // a G + G B
#pragma unroll
        for (int r = 0; r < kThinRows; ++r)
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int m = 0; m < S; ++m) g[r][j] = fmaf(x[r][m], t(m, j), g[r][j]);
    }
    // x holds X0: dU = (G - X0 <G, X0>) / |U|, or G / eps below eps
    float dot = 0.f;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) dot = fmaf(g[r][j], x[r][j], dot);
    dot = group_sum(dot, sh.group);
    if (norm < eps) dot = 0.f;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            if (live && l < sh.L)
                v_x[base + l * sh.row_step + j * sh.col_step] = from_f32<T>(fmaf(-x[r][j], dot, g[r][j]) / d);
        }
}

// Momentum, orthogonalisation and the parameters' step in one pass. Matrices of
// hidden rows are neither read nor written.
template <typename T, typename M, int S>
__global__ void __launch_bounds__(kThinThreads)
    thin_muon_kernel(ThinShape sh, const __grid_constant__ MuonTable tab, const OrthoCoefficients co, float eps) {
    const int lane = threadIdx.x & (sh.group - 1);
    const long long b = ((long long)blockIdx.x * kThinThreads + threadIdx.x) / sh.group;
    bool live = b < sh.batch;
    const int t = live ? muon_tensor_of(tab, b) : 0;
    live = live && muon_visible(tab, t, b);
    if (__ballot_sync(0xffffffffu, live) == 0u) return; // the whole warp has nothing to do
    const size_t base = live ? (size_t)(b - tab.first[t]) * sh.L * S : 0;
    const T *grad = static_cast<const T *>(tab.grad[t]);
    M *mom = static_cast<M *>(tab.momentum[t]);
    T *param = static_cast<T *>(tab.param[t]);
    float x[kThinRows][S];
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            x[r][j] = 0.f;
            if (live && l < sh.L) {
                const size_t at = base + l * sh.row_step + j * sh.col_step;
                const float g = to_f32(grad[at]);
                const float m = muon_momentum(g, to_f32(mom[at]), tab.one_minus_mu);
                mom[at] = from_f32<M>(m);
                x[r][j] = muon_update(g, m, tab.mu, tab.nesterov);
            }
        }
    const float norm = frobenius<S>(x, sh.group);
    const float d = norm < eps ? eps : norm;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] / d;
    thin_iterate<S>(x, co, sh.group);
    const float lr = tab.lr[t], decay = tab.decay[t];
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            if (live && l < sh.L) {
                const size_t at = base + l * sh.row_step + j * sh.col_step;
                param[at] = from_f32<T>(muon_param(to_f32(param[at]), x[r][j], lr, decay));
            }
        }
}

static ThinShape thin_shape(long long batch, int rows, int cols) {
    ThinShape sh;
    sh.batch = batch;
    sh.L = rows < cols ? cols : rows;
    sh.S = rows < cols ? rows : cols;
    sh.group = 1;
    while (sh.group * kThinRows < sh.L) sh.group *= 2;
    sh.row_step = rows < cols ? 1 : cols;
    sh.col_step = rows < cols ? cols : 1;
    return sh;
}

// Blocks of a launch, or 0 if the batch is too large for one grid.
static unsigned thin_blocks(const ThinShape &sh, int threads) {
    const int per_block = threads / sh.group;
    const long long n = (sh.batch + per_block - 1) / per_block;
    return n > 0x7fffffffll ? 0u : (unsigned)n;
}

template <typename F> static int with_short(int S, F f) {
    switch (S) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    default: return f(std::integral_constant<int, 4>());
    }
}
template <typename F> static int with_type(int dtype, F f) {
    if (dtype == kOrthoF32) return f(float());
    if (dtype == kOrthoBF16) return f(__nv_bfloat16());
    return f(__half());
}

int ortho_thin_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream) {
    const ThinShape sh = thin_shape(batch, rows, cols);
    const unsigned blocks = thin_blocks(sh, kThinThreads);
    if (blocks == 0) return set_error(kErrInvalidArgument, "orthogonalize: too many matrices");
    return with_type(dtype, [&](auto tv) {
        using T = decltype(tv);
        return with_short(sh.S, [&](auto s) {
            thin_fwd_kernel<T, s.value><<<blocks, kThinThreads, 0, stream>>>(sh, (const T *)x, (T *)y, co, eps);
            return check_launch("thin_fwd_kernel");
        });
    });
}

int ortho_thin_bwd(long long batch, int rows, int cols, int dtype, const void *x, const void *v_y, void *v_x,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream) {
    const ThinShape sh = thin_shape(batch, rows, cols);
    // 32 steps of 4 x 4 values for 64 threads: 128 KiB of shared memory at most
    const int threads = co.steps <= 8 ? kThinThreads : 64;
    const unsigned blocks = thin_blocks(sh, threads);
    if (blocks == 0) return set_error(kErrInvalidArgument, "orthogonalize: too many matrices");
    const size_t smem = (size_t)co.steps * kThinRows * sh.S * threads * sizeof(float);
    return with_type(dtype, [&](auto tv) {
        using T = decltype(tv);
        return with_short(sh.S, [&](auto s) {
            auto *kernel = thin_bwd_kernel<T, s.value>;
            if (smem > 48 * 1024 &&
                cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
                return check_launch("thin_bwd_kernel attributes");
            kernel<<<blocks, threads, smem, stream>>>(sh, (const T *)x, (const T *)v_y, (T *)v_x, co, eps);
            return check_launch("thin_bwd_kernel");
        });
    });
}

int ortho_thin_muon(const MuonTable &table, int rows, int cols, const OrthoCoefficients &co, float eps,
                    cudaStream_t stream) {
    const ThinShape sh = thin_shape(table.first[table.n], rows, cols);
    const unsigned blocks = thin_blocks(sh, kThinThreads);
    if (blocks == 0) return set_error(kErrInvalidArgument, "muon: too many matrices");
    return with_type(table.dtype, [&](auto tv) {
        using T = decltype(tv);
        return with_short(sh.S, [&](auto s) {
            if (table.state_dtype == table.dtype)
                thin_muon_kernel<T, T, s.value><<<blocks, kThinThreads, 0, stream>>>(sh, table, co, eps);
            else
                thin_muon_kernel<T, float, s.value><<<blocks, kThinThreads, 0, stream>>>(sh, table, co, eps);
            return check_launch("thin_muon_kernel");
        });
    });
}

} // namespace gsb
