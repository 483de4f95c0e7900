// Newton-Schulz orthogonalisation of matrices, its backward pass and the Muon
// step: the entry points, and the passes before and after the tiled products.
//
// Numbers of the tiled path. Every matrix of the iteration is kept as
// scale * (hi + lo), both fp16 (22 significand bits), with power-of-two scales
// from bounds on its values, so that nothing overflows and little is subnormal:
// X <= s_max, the largest singular value that the polynomials reach from [0, 1];
// A <= s_max^2; B <= max |b t + c t^2| over t <= s_max^2. The diagonals of A and B are kept
// apart in 32 bits: near convergence A is close to a multiple of the identity, and
// rounding its diagonal would cost more than all of its other entries together.
// With A = D + O (D diagonal) the products are
//     A A = O O + D O + O D + D D,   B X = O_B X + D_B X,
// and the terms with a diagonal are element-wise, in the epilogue.
// Products are of hi + lo, in three matrix products (lo lo is below 2^-22). Those of
// bfloat16 matrices (8 bits) are of hi alone, with its 11 bits, while X itself goes from
// step to step with hi and lo: a X + B X is where small singular values would lose theirs.
// The result is then 0.0005 to 0.001 off (2-norm), against the type's own rounding of 0.0017; sums are read out of the tensor
// cores before their truncation counts beside that (ortho_gemm.cuh), so that it holds for long sides too.
// float16 results would be off by three times their rounding that way, and backward passes by the
// sum of theirs, so they take hi + lo as float32 does; so do matrices of at most 128 x 128, whose
// calls are bound by latency.
#include <algorithm>
#include <cmath>

#include "ortho.cuh"

namespace gsb {

// --- norms and the split into planes ----------------------------------------
// These passes are bound by memory: four values to an access where the matrix allows it, and
// several accesses a thread on their way at once.
constexpr int kNormThreads = 256;
constexpr int kSplitTile = 64;

// What is read: x, or the Muon update of its matrix.
template <typename T, typename M, bool MUON> struct OrthoSource {
    const T *x; // or the gradient
    M *mom;
    float mu, one_minus_mu;
    int nesterov;
    using VT = typename Quad<T>::type;
    using VM = typename Quad<M>::type;

    __device__ __forceinline__ OrthoSource(const void *xs, const MuonTable &tab, int t, long long b, size_t numel) {
        if (MUON) {
            const size_t at = (size_t)(b - tab.first[t]) * numel;
            x = static_cast<const T *>(tab.grad[t]) + at;
            mom = static_cast<M *>(tab.momentum[t]) + at;
            mu = tab.mu;
            one_minus_mu = tab.one_minus_mu;
            nesterov = tab.nesterov;
        } else {
            x = static_cast<const T *>(xs) + (size_t)b * numel;
        }
    }
    __device__ __forceinline__ bool aligned() const {
        return reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 &&
               (!MUON || reinterpret_cast<uintptr_t>(mom) % (4 * sizeof(M)) == 0);
    }
    __device__ __forceinline__ float4 get4(size_t e, float4 &m) const {
        if (MUON) m = Quad<M>::get(*reinterpret_cast<const VM *>(mom + e));
        return Quad<T>::get(*reinterpret_cast<const VT *>(x + e));
    }
    __device__ __forceinline__ float get1(size_t e, float &m) const {
        if (MUON) m = to_f32(mom[e]);
        return to_f32(x[e]);
    }
    __device__ __forceinline__ float update(float g, float &m) const {
        if (!MUON) return g;
        m = muon_momentum(g, m, one_minus_mu);
        return muon_update(g, m, mu, nesterov);
    }
    __device__ __forceinline__ float4 update(float4 g, float4 &m) const {
        return make_float4(update(g.x, m.x), update(g.y, m.y), update(g.z, m.z), update(g.w, m.w));
    }
};

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kNormThreads / 32];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kNormThreads / 32; ++w) v += part[w];
    return v;
}

// Sums of squares of the chunks (a multiple of 4 values) of each matrix, in 64 bits and a fixed order.
template <typename T, typename M, bool MUON>
__global__ void __launch_bounds__(kNormThreads)
    ortho_norm_kernel(const void *x, const __grid_constant__ MuonTable tab, size_t numel, size_t chunk_size, int chunks,
                      double *partial, int *error) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0 && error) *error = 0; // nothing has waited yet
    const long long b = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks);
    const int t = MUON ? muon_tensor_of(tab, b) : 0;
    if (MUON && !muon_visible(tab, t, b)) return;
    const OrthoSource<T, M, MUON> src(x, tab, t, b, numel);
    const size_t first = (size_t)chunk * chunk_size, last = min(numel, first + chunk_size);
    const int quads = src.aligned() ? (int)((last - first) / 4) : 0;
    constexpr int U = 4;
    double s = 0.0;
    for (int i0 = threadIdx.x; i0 < quads; i0 += U * kNormThreads) {
        float4 g[U], m[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            g[u] = m[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + u * kNormThreads < quads) g[u] = src.get4(first + 4 * (size_t)(i0 + u * kNormThreads), m[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4 w = src.update(g[u], m[u]);
            s = fma((double)w.x, (double)w.x, s);
            s = fma((double)w.y, (double)w.y, s);
            s = fma((double)w.z, (double)w.z, s);
            s = fma((double)w.w, (double)w.w, s);
        }
    }
#pragma unroll 4
    for (size_t e = first + 4 * (size_t)quads + threadIdx.x; e < last; e += kNormThreads) {
        float m = 0.f;
        const float g = src.get1(e, m);
        const double v = src.update(g, m);
        s = fma(v, v, s);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double sum_partials(const double *partial, long long b, int chunks) {
    double s = 0.0;
    for (int c = threadIdx.x; c < chunks; c += kNormThreads) s += partial[b * chunks + c];
    return block_sum(s);
}

__device__ __forceinline__ uint2 pack4(float4 f) {
    return Quad<__half>::put(f);
}
// Four values to both planes; a row has room for whole fours (its length is rounded up to 8).
__device__ __forceinline__ void planes_put4(const OrthoPlanes &p, size_t at, float4 v) {
    const uint2 h = pack4(v);
    const float4 f = Quad<__half>::get(h);
    *reinterpret_cast<uint2 *>(p.hi + at) = h;
    *reinterpret_cast<uint2 *>(p.lo + at) = pack4(make_float4(v.x - f.x, v.y - f.y, v.z - f.z, v.w - f.w));
}
__device__ __forceinline__ float4 planes_get4(const OrthoPlanes &p, size_t at) {
    const float4 h = Quad<__half>::get(*reinterpret_cast<const uint2 *>(p.hi + at));
    const float4 l = Quad<__half>::get(*reinterpret_cast<const uint2 *>(p.lo + at));
    return make_float4(h.x + l.x, h.y + l.y, h.z + l.z, h.w + l.w);
}

// planes <- factor * source, in the orientation whose rows are the shorter side.
// eps > 0: factor = scale / max(norm, eps), and norm_out gets the norm, or -1
// below eps. eps = 0: factor = the power of two that brings the norm to (scale / 2, scale], and
// norm_out gets the factor. A block takes 64 x 64 values, a thread four rows of four.
template <typename T, typename M, bool MUON>
__global__ void __launch_bounds__(kNormThreads)
    ortho_split_kernel(const void *x, const __grid_constant__ MuonTable tab, int rows, int cols, int transposed,
                       const double *partial, int chunks, float scale, float eps, double *norm_out, OrthoPlanes out,
                       int tiles_r, int tiles_c) {
    __shared__ float tile[kSplitTile][kSplitTile + 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long per = (long long)tiles_r * tiles_c;
    const long long b = blockIdx.x / per;
    const int ti = (int)(blockIdx.x % per);
    const int r0 = (ti / tiles_c) * kSplitTile, c0 = (ti % tiles_c) * kSplitTile;
    const int t = MUON ? muon_tensor_of(tab, b) : 0;
    if (MUON && !muon_visible(tab, t, b)) return;
    const bool turned = MUON ? tab.transposed[t] : transposed;
    if (MUON && turned != (bool)transposed) { // the tensor of the other orientation: its own rows and columns
        const int k = rows;
        rows = cols;
        cols = k;
    }
    const int tr0 = MUON && turned != (bool)transposed ? c0 : r0, tc0 = MUON && turned != (bool)transposed ? r0 : c0;
    const OrthoSource<T, M, MUON> src(x, tab, t, b, (size_t)rows * cols);
    const bool quads = src.aligned() && cols % 4 == 0;
    const int q = threadIdx.x % 16 * 4, r = threadIdx.x / 16; // columns q .. q + 3 of rows r, r + 16, ..
    float4 g[4], m[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int row = tr0 + r + 16 * u, col = tc0 + q;
        const size_t e = (size_t)row * cols + col;
        g[u] = m[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row >= rows) continue;
        if (quads) {
            if (col < cols) g[u] = src.get4(e, m[u]);
        } else {
            if (col < cols) g[u].x = src.get1(e, m[u].x);
            if (col + 1 < cols) g[u].y = src.get1(e + 1, m[u].y);
            if (col + 2 < cols) g[u].z = src.get1(e + 2, m[u].z);
            if (col + 3 < cols) g[u].w = src.get1(e + 3, m[u].w);
        }
    }
    const double norm = sqrt(sum_partials(partial, b, chunks));
    float pre, div, mul;
    if (eps > 0.f) {
        const Divisor d = divisor_of(norm, eps);
        pre = d.pre;
        div = d.div;
        mul = scale;
        if (ti == 0 && threadIdx.x == 0) norm_out[b] = d.small ? -1.0 : norm;
    } else { // in two factors: their product may lie outside of a float's range
        const int e = norm > 0.0 && norm < (double)INFINITY ? ilogb(norm) + 1 : 0;
        pre = (float)ldexp(1.0, -(e / 2));
        div = 1.f;
        mul = (float)ldexp((double)scale, e / 2 - e);
        if (ti == 0 && threadIdx.x == 0) norm_out[b] = ldexp((double)scale, -e);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int row = tr0 + r + 16 * u, col = tc0 + q;
        if (row >= rows || col >= cols) continue;
        float4 w = src.update(g[u], m[u]);
        if (MUON) {
            M *to = src.mom + (size_t)row * cols + col;
            if (quads) {
                *reinterpret_cast<typename Quad<M>::type *>(to) = Quad<M>::put(m[u]);
            } else {
                to[0] = from_f32<M>(m[u].x);
                if (col + 1 < cols) to[1] = from_f32<M>(m[u].y);
                if (col + 2 < cols) to[2] = from_f32<M>(m[u].z);
                if (col + 3 < cols) to[3] = from_f32<M>(m[u].w);
            }
        }
        w = make_float4(w.x * pre / div * mul, w.y * pre / div * mul, w.z * pre / div * mul, w.w * pre / div * mul);
        if (!turned) {
            planes_put4(out, (size_t)b * out.stride + (size_t)row * out.ld + col, w);
        } else {
            float *to = &tile[r + 16 * u][q];
            to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
        }
    }
    if (!turned) return;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) { // the planes' rows are the tensor's columns
        const int k = r + 16 * u, row = tc0 + k, col = tr0 + q;
        if (row < cols && col < rows)
            planes_put4(out, (size_t)b * out.stride + (size_t)row * out.ld + col,
                        make_float4(tile[q][k], tile[q + 1][k], tile[q + 2][k], tile[q + 3][k]));
    }
}

// Partial sums of <G, X> over the rows of each matrix, eight values at a time in 64 bits.
__global__ void __launch_bounds__(kNormThreads)
    ortho_dot_kernel(OrthoPlanes g, OrthoPlanes x, int m, int n, int chunks, double *partial) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long b = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks);
    const int fours = (n + 3) / 4, rows = (m - chunk + chunks - 1) / chunks; // rows chunk, chunk + chunks, ..
    double s = 0.0;
#pragma unroll 4
    for (long long e = threadIdx.x; e < (long long)rows * fours; e += kNormThreads) {
        const int i = (int)(e / fours), j = 4 * (int)(e - (long long)i * fours);
        const size_t row = (size_t)(chunk + i * chunks);
        const float4 u = planes_get4(g, (size_t)b * g.stride + row * g.ld + j), v = planes_get4(x, (size_t)b * x.stride + row * x.ld + j);
        s = fma((double)u.x, (double)v.x, s);
        if (j + 1 < n) s = fma((double)u.y, (double)v.y, s);
        if (j + 2 < n) s = fma((double)u.z, (double)v.z, s);
        if (j + 3 < n) s = fma((double)u.w, (double)v.w, s);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// G's planes brought back to a norm in (scale / 2, scale] by a power of two, which its
// factor takes too. <G, G> in `partial`.
__global__ void __launch_bounds__(kNormThreads)
    ortho_rescale_kernel(OrthoPlanes g, int m, int n, int chunks, const double *partial, float scale, const double *factor_in,
                         float fallen, double *factor_out) {
    const long long b = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks);
    const float norm = (float)sqrt(sum_partials(partial, b, chunks));
    const int e = norm > 0.f && norm < INFINITY ? min(max(ilogb(norm) + 1, -100), 126) : ilogb(scale);
    const float mul = scale * exp2f((float)-e);
    if (chunk == 0 && threadIdx.x == 0) factor_out[b] = factor_in[b] * (double)fallen * (double)mul;
    for (int i = chunk; i < m; i += chunks)
        for (int j = threadIdx.x; j < n; j += kNormThreads) {
            const size_t at = (size_t)b * g.stride + (size_t)i * g.ld + j;
            const float v = (__half2float(g.hi[at]) + __half2float(g.lo[at])) * mul;
            const __half h = __float2half_rn(v);
            g.hi[at] = h;
            g.lo[at] = __float2half_rn(v - __half2float(h));
        }
}

// v_x = (G - X0 <G, X0>) / norm, or G / eps for a matrix whose norm is below eps.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
    ortho_grad_out_kernel(OrthoPlanes g, OrthoPlanes x, int rows, int cols, int transposed, const double *partial,
                          int chunks, const double *norms, const double *g_factor, float g_scale, float x_scale, float eps,
                          T *v_x, int tiles_r, int tiles_c, const int *error, const int *kept_error) {
    __shared__ float tile[kSplitTile][kSplitTile + 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long per = (long long)tiles_r * tiles_c;
    const long long b = blockIdx.x / per;
    const int ti = (int)(blockIdx.x % per);
    const int i0 = (ti / tiles_c) * kSplitTile, j0 = (ti % tiles_c) * kSplitTile; // of the planes
    const int m = transposed ? cols : rows, n = transposed ? rows : cols;
    const int q = threadIdx.x % 16 * 4, r = threadIdx.x / 16;
    float4 gv[4], xv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = i0 + r + 16 * u, j = j0 + q;
        if (i < m && j < n) {
            gv[u] = planes_get4(g, (size_t)b * g.stride + (size_t)i * g.ld + j);
            xv[u] = planes_get4(x, (size_t)b * x.stride + (size_t)i * x.ld + j);
        }
    }
    const double dot = sum_partials(partial, b, chunks);
    const double norm = norms[b], factor = g_factor[b];
    const bool small = norm < 0.0;
    const float along = small ? 0.f : (float)(dot / ((double)x_scale * x_scale));
    const double by = small ? (double)eps : norm;
    // in 32 bits, one after the other (the factor and g_scale are powers of two), where that keeps all in range; else in 64
    const bool middle = by > 0x1p-100 && by < 0x1p120 && factor >= 0x1p-112 && factor <= 0x1p114;
    const float div = (float)by, f = (float)factor;
    const double all = 1.0 / ((double)g_scale * factor * by);
    const bool poisoned = *error != 0 || (kept_error && *kept_error != 0);
    auto value = [&](float gw, float xw) {
        const float v = fmaf(-xw, along, gw);
        return poisoned ? NAN : middle ? v / g_scale / f / div : (float)((double)v * all);
    };
    T *out = v_x + (size_t)b * rows * cols;
    const bool quads = cols % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0;
    auto put = [&](int row, int col, float4 v) {
        T *to = out + (size_t)row * cols + col;
        if (quads) {
            *reinterpret_cast<typename Quad<T>::type *>(to) = Quad<T>::put(v);
        } else {
            to[0] = from_f32<T>(v.x);
            if (col + 1 < cols) to[1] = from_f32<T>(v.y);
            if (col + 2 < cols) to[2] = from_f32<T>(v.z);
            if (col + 3 < cols) to[3] = from_f32<T>(v.w);
        }
    };
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = i0 + r + 16 * u, j = j0 + q;
        if (i >= m || j >= n) continue;
        const float4 v = make_float4(value(gv[u].x, xv[u].x), value(gv[u].y, xv[u].y), value(gv[u].z, xv[u].z),
                                     value(gv[u].w, xv[u].w));
        if (!transposed) {
            put(i, j, v);
        } else {
            float *to = &tile[r + 16 * u][q];
            to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
        }
    }
    if (!transposed) return;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int k = r + 16 * u, row = j0 + k, col = i0 + q; // of v_x
        if (row < rows && col < cols) put(row, col, make_float4(tile[q][k], tile[q + 1][k], tile[q + 2][k], tile[q + 3][k]));
    }
}

// --- the plan of one call -----------------------------------------------------
constexpr double kPlaneTop = 16384.0; // bound on scaled values: a factor of four below fp16's largest

static double pow2_floor(double v) { return std::exp2(std::floor(std::log2(v))); }

struct OrthoScales {
    double x, a, b;           // of X, A, B
    double top, top_b, slope; // bounds: singular values, |B|, |p'|
    double worst_t;           // |b| 2 top + 4 |c| top^3 over the steps: of T for a G of norm 1
};

// Bounds over [0, 1] under the steps' polynomials p(s) = a s + b s^3 + c s^5.
static OrthoScales ortho_scales(const OrthoCoefficients &co) {
    OrthoScales r = {};
    double m = 1.0, top = 1.0;
    r.slope = 1.0;
    for (int k = 0; k < co.steps; ++k) {
        const double a = co.c[k][0], b = co.c[k][1], c = co.c[k][2];
        auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
        auto dp = [&](double t) { return std::fabs(a + t * (3 * b + t * 5 * c)); }; // t = s^2
        auto q = [&](double t) { return std::fabs(t * (b + t * c)); };
        double next = p(m), slope = std::fmax(dp(0.0), dp(m * m)), qb = q(m * m);
        // interior extrema: p' = 0 at t = (-3b +- sqrt(9 b^2 - 20 a c)) / (10 c); p'' = 0 at t = -3b / (10 c); q' = 0 at -b / 2c
        auto at = [&](double t) { if (t > 0 && t < m * m) next = std::fmax(next, p(std::sqrt(t))); };
        if (c != 0.0) {
            const double disc = 9 * b * b - 20 * a * c;
            if (disc >= 0) {
                at((-3 * b + std::sqrt(disc)) / (10 * c));
                at((-3 * b - std::sqrt(disc)) / (10 * c));
            }
            const double ti = -3 * b / (10 * c), tq = -b / (2 * c);
            if (ti > 0 && ti < m * m) slope = std::fmax(slope, dp(ti));
            if (tq > 0 && tq < m * m) qb = std::fmax(qb, q(tq));
        } else if (b != 0.0) {
            at(-a / (3 * b));
        }
        r.slope = std::fmax(r.slope, slope);
        r.top_b = std::fmax(r.top_b, qb);
        r.worst_t = std::fmax(r.worst_t, 2 * m * (std::fabs(b) + 2 * std::fabs(c) * m * m));
        m = next;
        top = std::fmax(top, m);
    }
    r.top = top;
    return r;
}

constexpr double kOrthoMaxTop = 16.0; // larger singular values would leave the planes' range

struct OrthoPlan {
    int rows, cols, m, n, transposed, steps;
    bool split;
    int chunks;        // of the norm's sum
    size_t chunk_size; // values
    OrthoScales s;
    int ldx, lda;
    long long px, pa; // elements of one matrix's plane
    size_t per_matrix, fixed;       // scratch bytes: a matrix's, and for alignment
    size_t kept_matrix, kept_fixed; // of the state that a backward pass needs
};

static size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

static OrthoPlan ortho_plan(int rows, int cols, int dtype, const OrthoCoefficients &co, bool backward, bool kept) {
    OrthoPlan p = {};
    p.rows = rows;
    p.cols = cols;
    p.transposed = rows > cols;
    p.m = p.transposed ? cols : rows;
    p.n = p.transposed ? rows : cols;
    p.steps = co.steps;
    p.split = dtype != kOrthoBF16 || backward || kept || p.n <= 128;
    const size_t numel = (size_t)rows * cols;
    p.chunk_size = std::max<size_t>(8192, (numel / 512 + 3) / 4 * 4); // about 512 blocks for a large matrix
    p.chunks = (int)((numel + p.chunk_size - 1) / p.chunk_size);
    p.s = ortho_scales(co);
    p.ldx = (p.n + 7) / 8 * 8;
    p.lda = (p.m + 7) / 8 * 8;
    p.px = (long long)p.m * p.ldx;
    p.pa = (long long)p.m * p.lda;
    const size_t halves = 2 * sizeof(__half);
    p.kept_matrix = co.steps * (halves * (p.px + 2 * p.pa) + 2 * sizeof(float) * p.m) + sizeof(double);
    p.kept_fixed = 256 * (size_t)(8 * co.steps + 2);
    size_t bytes = sizeof(double) * (size_t)(p.chunks + 2); // sums, and norms or two factors
    if (backward)
        bytes += 2 * halves * (p.px + p.pa); // G twice, S, T
    else if (!kept) // else all but the sums lies in the state
        bytes += 2 * halves * (p.px + p.pa) + 2 * sizeof(float) * p.m; // X twice, A, B, diagonals
    p.per_matrix = bytes;
    p.fixed = 256 * 24;
    if (backward && !kept) {
        p.per_matrix += p.kept_matrix;
        p.fixed += p.kept_fixed;
    }
    return p;
}

constexpr size_t kScratchBudget = (size_t)1 << 30;

static long long ortho_chunk(const OrthoPlan &p, long long batch) {
    long long n = (long long)(kScratchBudget / p.per_matrix);
    // one launch's grid holds a chunk's tiles
    const long long tiles = (long long)((p.rows + 63) / 64) * ((p.cols + 63) / 64) + p.chunks;
    if (n > 0x3fffffffll / tiles) n = 0x3fffffffll / tiles;
    if (n < 1) n = 1;
    return n < batch ? n : batch;
}

struct Carver {
    char *p;
    template <typename T> T *take(size_t n) {
        T *r = reinterpret_cast<T *>(p);
        p += align256(n * sizeof(T));
        return r;
    }
    OrthoPlanes planes(long long batch, long long size, int ld) {
        OrthoPlanes o;
        o.hi = take<__half>((size_t)batch * size);
        o.lo = take<__half>((size_t)batch * size);
        o.ld = ld;
        o.stride = size;
        return o;
    }
};

// What a backward pass needs of the steps: each one's X, A and B, and the norms. A wait of the steps that ran out is known by
// the error word of tiled products, by NaN in the place of its matrix's norm of the clustered kernel, which leaves the word alone.
struct OrthoBuffers {
    int *error;
    OrthoPlanes x[kOrthoMaxSteps], a[kOrthoMaxSteps], b[kOrthoMaxSteps];
    float *da[kOrthoMaxSteps], *db[kOrthoMaxSteps];
    double *norms;

    OrthoBuffers(Carver &ws, const OrthoPlan &p, long long nb) {
        error = ws.take<int>(1);
        for (int k = 0; k < p.steps; ++k) {
            x[k] = ws.planes(nb, p.px, p.ldx);
            a[k] = ws.planes(nb, p.pa, p.lda);
            b[k] = ws.planes(nb, p.pa, p.lda);
            da[k] = ws.take<float>((size_t)nb * p.m);
            db[k] = ws.take<float>((size_t)nb * p.m);
        }
        norms = ws.take<double>(nb);
    }
};

// f(T, M, is it a Muon step)
template <typename F> static int with_source(int dtype, const MuonTable &tab, F f) {
    using std::false_type;
    using std::true_type;
    if (tab.n == 0) {
        if (dtype == kOrthoF32) return f(float(), float(), false_type());
        if (dtype == kOrthoBF16) return f(__nv_bfloat16(), float(), false_type());
        return f(__half(), float(), false_type());
    }
    if (tab.dtype == kOrthoF32) return f(float(), float(), true_type());
    if (tab.dtype == kOrthoBF16)
        return tab.state_dtype == kOrthoF32 ? f(__nv_bfloat16(), float(), true_type()) : f(__nv_bfloat16(), __nv_bfloat16(), true_type());
    return tab.state_dtype == kOrthoF32 ? f(__half(), float(), true_type()) : f(__half(), __half(), true_type());
}

static int run_split(const OrthoPlan &p, long long nb, const void *x, int dtype, const MuonTable &tab, float scale, float eps,
                     double *norm_out, double *partial, const OrthoPlanes &out, int *error, cudaStream_t stream) {
    return with_source(dtype, tab, [&](auto tv, auto mv, auto muon) {
        using T = decltype(tv);
        using M = decltype(mv);
        constexpr bool kMuon = decltype(muon)::value;
        // the call's first launch (it resets the error word) follows the stream's order in full: what a launch before it did not
        // wait for may be our input
        const auto blocks = (unsigned)(nb * p.chunks);
        const size_t numel = (size_t)p.rows * p.cols;
        if (error) {
            ortho_norm_kernel<T, M, kMuon><<<blocks, kNormThreads, 0, stream>>>(x, tab, numel, p.chunk_size, p.chunks, partial, error);
            if (int e = check_launch("ortho_norm_kernel")) return e;
        } else if (int e = launch_after(ortho_norm_kernel<T, M, kMuon>, blocks, kNormThreads, 0, stream, "ortho_norm_kernel", x, tab, numel,
                                        p.chunk_size, p.chunks, partial, error)) {
            return e;
        }
        const int tr = (p.rows + kSplitTile - 1) / kSplitTile, tc = (p.cols + kSplitTile - 1) / kSplitTile;
        return launch_after(ortho_split_kernel<T, M, kMuon>, (unsigned)(nb * tr * tc), kNormThreads, 0, stream, "ortho_split_kernel",
                            x, tab, p.rows, p.cols, p.transposed, (const double *)partial, p.chunks, scale, eps, norm_out, out, tr, tc);
    });
}

static int run_dot(const OrthoPlan &p, long long nb, const OrthoPlanes &g, const OrthoPlanes &x, double *partial, cudaStream_t stream) {
    return launch_after(ortho_dot_kernel, (unsigned)(nb * p.chunks), kNormThreads, 0, stream, "ortho_dot_kernel", g, x, p.m, p.n, p.chunks,
                        partial);
}

static OrthoGemm gemm_base(const OrthoPlan &p, long long nb, int *error) {
    OrthoGemm g = {};
    g.error = error;
    g.batch = nb;
    g.pairs = 1;
    g.split = p.split;
    g.transposed = p.transposed;
    return g;
}

// A and its polynomial B of step k, from X_k.
static int run_poly(const OrthoPlan &p, long long nb, const float c[3], double sb, const OrthoPlanes &x,
                    const OrthoPlanes &a, const OrthoPlanes &b, float *da, float *db, const MuonTable *tab,
                    int *error, cudaStream_t stream) {
    OrthoGemm g = gemm_base(p, nb, error);
    g.M = g.N = p.m;
    g.K = p.n;
    g.q_k_major = g.symmetric = 1;
    g.p[0] = g.q[0] = x;
    g.epilogue = kEpiGram;
    g.c[0] = (float)(p.s.a / (p.s.x * p.s.x));
    g.c[1] = (float)(1.0 / (p.s.x * p.s.x));
    g.out = a;
    g.diag_out = da;
    if (int e = ortho_gemm(g, tab, stream)) return e;
    g.K = p.m;
    g.p[0] = g.q[0] = g.e = a;
    g.epilogue = kEpiSquare;
    g.c[0] = (float)(c[1] * sb / p.s.a);
    g.c[1] = (float)(c[2] * sb / p.s.a);
    g.c[2] = (float)(c[2] * sb / (p.s.a * p.s.a));
    g.c[3] = c[1];
    g.c[4] = c[2];
    g.c[5] = (float)(c[2] / (p.s.a * p.s.a));
    g.out = b;
    g.diag_in = da;
    g.diag_out = db;
    return ortho_gemm(g, tab, stream);
}

static OrthoGemm apply_gemm(const OrthoPlan &p, long long nb, float a, double sb, const OrthoPlanes &x,
                            const OrthoPlanes &b, const float *db, int *error) {
    OrthoGemm g = gemm_base(p, nb, error);
    g.M = g.K = p.m;
    g.N = p.n;
    g.p[0] = b;
    g.q[0] = g.e = x;
    g.diag_in = db;
    g.epilogue = kEpiApply;
    g.c[0] = a;
    g.c[1] = (float)(1.0 / sb);
    g.c[2] = 1.f;
    return g;
}

static int ortho_tiled_fwd(const OrthoPlan &p, const OrthoCoefficients &co, long long nb, const void *src,
                           void *y, int dtype, const MuonTable &tab, float eps, char *scratch, cudaStream_t stream) {
    Carver ws{scratch};
    OrthoPlanes x[2] = {ws.planes(nb, p.px, p.ldx), ws.planes(nb, p.px, p.ldx)};
    const OrthoPlanes a = ws.planes(nb, p.pa, p.lda), b = ws.planes(nb, p.pa, p.lda);
    float *da = ws.take<float>((size_t)nb * p.m), *db = ws.take<float>((size_t)nb * p.m);
    double *partial = ws.take<double>((size_t)nb * p.chunks);
    double *norms = ws.take<double>(nb);
    int *error = ws.take<int>(1);
    const MuonTable *t = tab.n > 0 ? &tab : nullptr;
    if (int e = run_split(p, nb, src, dtype, tab, (float)p.s.x, eps, norms, partial, x[0], error, stream)) return e;
    for (int k = 0; k < co.steps; ++k) {
        const OrthoPlanes &from = x[k & 1];
        if (int e = run_poly(p, nb, co.c[k], p.s.b, from, a, b, da, db, t, error, stream)) return e;
        OrthoGemm g = apply_gemm(p, nb, co.c[k][0], p.s.b, from, b, db, error);
        if (k + 1 < co.steps) {
            g.out = x[(k + 1) & 1];
        } else {
            g.epilogue = t ? kEpiMuon : kEpiOut;
            g.c[2] = (float)(1.0 / p.s.x);
            g.y = y;
            g.dtype = dtype;
        }
        if (int e = ortho_gemm(g, t, stream)) return e;
    }
    return kOk;
}

// B's scale where the backward pass reads it. There both products of G's step accumulate together: (B's scale)
// (G's) = (T's)(X's). With |G| scaled to at most kPlaneTop, T's scaled bound is worst_t kPlaneTop sb / sx.
static double backward_scale(const OrthoPlan &p) { return std::fmin(p.s.b, pow2_floor(p.s.x / p.s.worst_t)); }

// The steps, each one's X, A and B kept; y may be NULL (the last product is then left out).
static int ortho_tiled_kept(const OrthoPlan &p, const OrthoCoefficients &co, long long nb, const void *src, void *y, int dtype,
                            const OrthoBuffers &w, float eps, double *partial, cudaStream_t stream) {
    int *const error = w.error;
    const double sb = backward_scale(p);
    const MuonTable none = {};
    if (int e = run_split(p, nb, src, dtype, none, (float)p.s.x, eps, w.norms, partial, w.x[0], error, stream)) return e;
    for (int k = 0; k < co.steps; ++k) {
        if (int e = run_poly(p, nb, co.c[k], sb, w.x[k], w.a[k], w.b[k], w.da[k], w.db[k], nullptr, error, stream)) return e;
        OrthoGemm g = apply_gemm(p, nb, co.c[k][0], sb, w.x[k], w.b[k], w.db[k], error);
        if (k + 1 < co.steps) {
            g.out = w.x[k + 1];
        } else if (y) {
            g.epilogue = kEpiOut;
            g.c[2] = (float)(1.0 / p.s.x);
            g.y = y;
            g.dtype = dtype;
        } else {
            break;
        }
        if (int e = ortho_gemm(g, nullptr, stream)) return e;
    }
    return kOk;
}

// Back through the steps, kept by the forward pass or taken again here:
//     S = G X^T + X G^T,  T = b S + c (S A + A S),  G <- a G + B G + T X.
// G's scale falls by the power of two above the largest slope |p'| at each
// step, which bounds how far its norm can grow; it is measured anew before
// that has cost it its low bits.
static int ortho_tiled_bwd(const OrthoPlan &p, const OrthoCoefficients &co, long long nb, const void *src,
                           const void *v, void *v_x, int dtype, float eps, void *kept, char *scratch, cudaStream_t stream) {
    const int K = co.steps;
    Carver ws{scratch}, own{static_cast<char *>(kept)};
    const OrthoBuffers w(kept ? own : ws, p, nb);
    OrthoPlanes gr[2] = {ws.planes(nb, p.px, p.ldx), ws.planes(nb, p.px, p.ldx)};
    const OrthoPlanes s = ws.planes(nb, p.pa, p.lda), t = ws.planes(nb, p.pa, p.lda);
    double *partial = ws.take<double>((size_t)nb * p.chunks);
    double *factor[2] = {ws.take<double>(nb), ws.take<double>(nb)};
    double *const norms = w.norms;
    int *error = kept ? ws.take<int>(1) : w.error;
    const MuonTable none = {};
    const double shrink = std::exp2(std::ceil(std::log2(p.s.slope)));
    const double sb = backward_scale(p);
    if (!kept)
        if (int e = ortho_tiled_kept(p, co, nb, src, nullptr, dtype, w, eps, partial, stream)) return e;
    if (int e = run_split(p, nb, v, dtype, none, (float)kPlaneTop, 0.f, factor[0], partial, gr[K & 1], kept ? error : nullptr, stream))
        return e;
    double grown = 1.0; // G's scale has fallen by this
    for (int k = K - 1; k >= 0; --k) {
        const OrthoPlanes &from = gr[(k + 1) & 1], &to = gr[k & 1];
        // scaled G is at most kPlaneTop, so S is at most 2 top kPlaneTop sx before its own scale
        const double ss = pow2_floor(1.0 / (2.0 * p.s.top));      // S's scale for G's scaled values
        const double st = sb / p.s.x;                             // T's
        OrthoGemm g = gemm_base(p, nb, error);
        g.pairs = 2;
        g.M = g.N = p.m;
        g.K = p.n;
        g.q_k_major = g.symmetric = 1;
        g.p[0] = g.q[1] = from;
        g.q[0] = g.p[1] = w.x[k];
        g.epilogue = kEpiSym;
        g.c[0] = (float)(ss / p.s.x);
        g.out = s;
        if (int e = ortho_gemm(g, nullptr, stream)) return e;
        g.K = p.m;
        g.p[0] = g.q[1] = g.e = s;
        g.q[0] = g.p[1] = w.a[k];
        g.epilogue = kEpiAnti;
        g.diag_in = w.da[k];
        g.c[0] = (float)(co.c[k][1] * st / ss);
        g.c[1] = (float)(co.c[k][2] * st / ss);
        g.c[2] = (float)(co.c[k][2] * st / (ss * p.s.a));
        g.out = t;
        if (int e = ortho_gemm(g, nullptr, stream)) return e;
        OrthoGemm h = apply_gemm(p, nb, co.c[k][0], sb, from, w.b[k], w.db[k], error);
        h.pairs = 2;
        h.p[1] = t;
        h.q[1] = w.x[k];
        h.c[2] = (float)(1.0 / shrink);
        h.out = to;
        if (int e = ortho_gemm(h, nullptr, stream)) return e;
        grown /= shrink;
        if (grown < 1.0 / 256 && k > 0) { // the bound is far off by now: measure the norm
            if (int e = run_dot(p, nb, to, to, partial, stream)) return e;
            ortho_rescale_kernel<<<(unsigned)(nb * p.chunks), kNormThreads, 0, stream>>>(
                to, p.m, p.n, p.chunks, partial, (float)kPlaneTop, factor[0], (float)grown, factor[1]);
            if (int e = check_launch("ortho_rescale_kernel")) return e;
            std::swap(factor[0], factor[1]);
            grown = 1.0;
        }
    }
    if (int e = run_dot(p, nb, gr[0], w.x[0], partial, stream)) return e;
    const int tr = (p.m + kSplitTile - 1) / kSplitTile, tc = (p.n + kSplitTile - 1) / kSplitTile;
    const int *kept_error = kept && !ortho_is_clustered(p.rows, p.cols) ? w.error : nullptr;
    return with_source(dtype, none, [&](auto tv, auto, auto) {
        using T = decltype(tv);
        return launch_after(ortho_grad_out_kernel<T>, (unsigned)(nb * tr * tc), kNormThreads, 0, stream, "ortho_grad_out_kernel", gr[0],
                            w.x[0], p.rows, p.cols, p.transposed, (const double *)partial, p.chunks, (const double *)norms,
                            (const double *)factor[0], (float)grown, (float)p.s.x, eps, static_cast<T *>(v_x), tr, tc, (const int *)error, kept_error);
    });
}

static int check_common(const char *what, long long batch, int rows, int cols, int dtype, int steps,
                        const float *coefficients, float eps, OrthoCoefficients *co) {
    if (batch < 0 || rows < 0 || cols < 0) return set_error(kErrInvalidArgument, "%s: negative size", what);
    if (std::max(rows, cols) > kOrthoMaxSide)
        return set_error(kErrInvalidArgument, "%s: [%d, %d]: a side may have %d values", what, rows, cols, kOrthoMaxSide);
    if (dtype < kOrthoF32 || dtype > kOrthoF16) return set_error(kErrUnsupported, "%s: dtype %d", what, dtype);
    if (steps < 1 || steps > kOrthoMaxSteps)
        return set_error(kErrInvalidArgument, "%s: steps must be 1 to %d, got %d", what, kOrthoMaxSteps, steps);
    if (coefficients == nullptr) return set_error(kErrInvalidArgument, "%s: no coefficients", what);
    if (!(eps > 0.f)) return set_error(kErrInvalidArgument, "%s: eps must be positive", what);
    co->steps = steps;
    for (int k = 0; k < steps; ++k)
        for (int j = 0; j < 3; ++j) {
            co->c[k][j] = coefficients[3 * k + j];
            if (!std::isfinite(co->c[k][j])) return set_error(kErrInvalidArgument, "%s: coefficient not finite", what);
        }
    const OrthoScales s = ortho_scales(*co);
    if (!(s.top <= kOrthoMaxTop))
        return set_error(kErrInvalidArgument, "%s: the polynomials take a singular value of 1 or less to %g; at most %g is held",
                         what, s.top, kOrthoMaxTop);
    return kOk;
}

static void finish_scales(OrthoPlan *p) {
    OrthoScales &s = p->s;
    s.x = pow2_floor(kPlaneTop / s.top);
    s.a = pow2_floor(kPlaneTop / (s.top * s.top));
    s.b = pow2_floor(kPlaneTop / std::fmax(s.top_b, 1.0));
}

static OrthoPlan make_plan(int rows, int cols, int dtype, const OrthoCoefficients &co, bool backward, bool kept) {
    OrthoPlan p = ortho_plan(rows, cols, dtype, co, backward, kept);
    finish_scales(&p);
    return p;
}

static size_t plan_bytes(const OrthoPlan &p, long long batch) {
    return (size_t)ortho_chunk(p, batch) * p.per_matrix + p.fixed;
}

} // namespace gsb

using namespace gsb;

extern "C" size_t gsb_orthogonalize_kept_bytes(long long batch, int rows, int cols, int steps) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || std::max(rows, cols) > kOrthoMaxSide || steps < 1 || steps > kOrthoMaxSteps ||
        ortho_is_thin(rows, cols))
        return 0;
    OrthoCoefficients co = {};
    co.steps = steps;
    const OrthoPlan p = ortho_plan(rows, cols, kOrthoF32, co, true, true);
    // the whole batch at once, or nothing
    if ((size_t)batch > kScratchBudget / (p.kept_matrix + p.per_matrix) || ortho_chunk(p, batch) < batch) return 0;
    return (size_t)batch * p.kept_matrix + p.kept_fixed;
}

extern "C" size_t gsb_orthogonalize_scratch_bytes(long long batch, int rows, int cols, int dtype, int steps, int backward, int kept) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || std::max(rows, cols) > kOrthoMaxSide || steps < 1 || steps > kOrthoMaxSteps ||
        ortho_is_thin(rows, cols))
        return 0;
    if (!backward && ortho_is_clustered(rows, cols)) return 0;
    OrthoCoefficients co = {};
    co.steps = steps;
    return plan_bytes(ortho_plan(rows, cols, dtype, co, backward != 0, kept != 0), batch);
}

static int check_kept(long long batch, int rows, int cols, int steps, const void *kept, size_t kept_bytes) {
    if (kept == nullptr) return kOk;
    const size_t needed = gsb_orthogonalize_kept_bytes(batch, rows, cols, steps);
    if (needed == 0) return set_error(kErrInvalidArgument, "orthogonalize: no state is kept of %lld x [%d, %d]", batch, rows, cols);
    if (kept_bytes < needed) return set_error(kErrInvalidArgument, "orthogonalize: the kept state needs %zu bytes", needed);
    return kOk;
}

extern "C" int gsb_orthogonalize_tile(long long batch, int rows, int cols, int dtype, int kept, int product, int sms) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || std::max(rows, cols) > kOrthoMaxSide || product < 0 || product > 5 || sms < 2 || ortho_is_thin(rows, cols) ||
        (product < 3 && ortho_is_clustered(rows, cols)))
        return 0;
    OrthoCoefficients co = {};
    co.steps = 1;
    const OrthoPlan p = ortho_plan(rows, cols, dtype, co, product >= 3, kept != 0);
    static const int epilogues[6] = {kEpiGram, kEpiSquare, kEpiApply, kEpiSym, kEpiAnti, kEpiApply};
    OrthoGemm g = gemm_base(p, batch, nullptr);
    g.M = p.m;
    g.N = product % 3 == 2 ? p.n : p.m;
    g.K = product % 3 == 0 ? p.n : p.m;
    g.pairs = product < 3 ? 1 : 2;
    g.epilogue = epilogues[product];
    g.symmetric = product % 3 != 2;
    const OrthoTile t = ortho_tile(g, sms);
    return 1000 * t.ranks + t.columns;
}

// What a kernel would follow: the caller's tensors, on a value's boundary, and memory that is read 16 bytes at a time.
static int check_tensor(const char *what, const void *p, int dtype) {
    if (p == nullptr) return set_error(kErrInvalidArgument, "%s: a tensor is missing", what);
    if (reinterpret_cast<uintptr_t>(p) % (dtype == kOrthoF32 ? 4 : 2))
        return set_error(kErrInvalidArgument, "%s: a tensor between two of its type's values", what);
    return kOk;
}
static int check_room(const char *what, const void *p) {
    if (reinterpret_cast<uintptr_t>(p) % 16) return set_error(kErrInvalidArgument, "%s: scratch and kept state are aligned to 16 bytes", what);
    return kOk;
}

static const char *at_matrix(const void *p, long long b, int rows, int cols, int dtype) {
    return static_cast<const char *>(p) + (size_t)b * rows * cols * (dtype == kOrthoF32 ? 4 : 2);
}

extern "C" int gsb_orthogonalize_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y, int steps,
                                     const float *coefficients, float eps, void *kept, size_t kept_bytes, void *scratch,
                                     size_t scratch_bytes, cudaStream_t stream) {
    OrthoCoefficients co = {};
    if (int e = check_common("orthogonalize", batch, rows, cols, dtype, steps, coefficients, eps, &co)) return e;
    if (batch == 0 || rows == 0 || cols == 0) return kOk;
    if (int e = check_kept(batch, rows, cols, steps, kept, kept_bytes)) return e;
    const size_t needed = gsb_orthogonalize_scratch_bytes(batch, rows, cols, dtype, steps, 0, kept != nullptr);
    if (needed > 0 && (scratch == nullptr || scratch_bytes < needed))
        return set_error(kErrInvalidArgument, "orthogonalize: %zu scratch bytes are needed", needed);
    if (int e = check_room("orthogonalize", needed > 0 ? scratch : nullptr)) return e;
    if (int e = check_room("orthogonalize", kept)) return e;
    for (const void *t : {x, (const void *)y})
        if (int e = check_tensor("orthogonalize", t, dtype)) return e;
    if (ortho_is_thin(rows, cols)) return ortho_thin_fwd(batch, rows, cols, dtype, x, y, co, eps, stream);
    const OrthoPlan p = make_plan(rows, cols, dtype, co, false, kept != nullptr);
    Carver own{static_cast<char *>(kept)};
    if (ortho_is_clustered(rows, cols)) {
        if (!kept)
            return ortho_cluster_fwd(batch, rows, cols, dtype, x, y, co, (float)p.s.x, (float)p.s.a, (float)p.s.b, eps, ClusterKept{}, stream);
        const OrthoBuffers w(own, p, batch);
        ClusterKept k = {};
        k.x = w.x[0], k.a = w.a[0], k.b = w.b[0];
        k.da = w.da[0], k.db = w.db[0], k.norms = w.norms;
        k.step = steps > 1 ? w.x[1].hi - w.x[0].hi : 0;
        return ortho_cluster_fwd(batch, rows, cols, dtype, x, y, co, (float)p.s.x, (float)p.s.a, (float)backward_scale(p), eps, k, stream);
    }
    if (kept) {
        const OrthoBuffers w(own, p, batch);
        Carver ws{static_cast<char *>(scratch)};
        return ortho_tiled_kept(p, co, batch, x, y, dtype, w, eps, ws.take<double>((size_t)batch * p.chunks), stream);
    }
    const long long chunk = ortho_chunk(p, batch);
    const MuonTable none = {};
    for (long long b = 0; b < batch; b += chunk) {
        if (int e = ortho_tiled_fwd(p, co, std::min(chunk, batch - b), at_matrix(x, b, rows, cols, dtype),
                                    const_cast<char *>(at_matrix(y, b, rows, cols, dtype)), dtype, none, eps,
                                    static_cast<char *>(scratch), stream))
            return e;
    }
    return kOk;
}

extern "C" int gsb_orthogonalize_bwd(long long batch, int rows, int cols, int dtype, const void *x, const void *v_y,
                                     void *v_x, int steps, const float *coefficients, float eps, void *kept, size_t kept_bytes,
                                     void *scratch, size_t scratch_bytes, cudaStream_t stream) {
    OrthoCoefficients co = {};
    if (int e = check_common("orthogonalize", batch, rows, cols, dtype, steps, coefficients, eps, &co)) return e;
    if (batch == 0 || rows == 0 || cols == 0) return kOk;
    if (int e = check_kept(batch, rows, cols, steps, kept, kept_bytes)) return e;
    const size_t needed = gsb_orthogonalize_scratch_bytes(batch, rows, cols, dtype, steps, 1, kept != nullptr);
    if (needed > 0 && (scratch == nullptr || scratch_bytes < needed))
        return set_error(kErrInvalidArgument, "orthogonalize: %zu scratch bytes are needed", needed);
    if (int e = check_room("orthogonalize", needed > 0 ? scratch : nullptr)) return e;
    if (int e = check_room("orthogonalize", kept)) return e;
    for (const void *t : {x, v_y, (const void *)v_x})
        if (int e = check_tensor("orthogonalize", t, dtype)) return e;
    if (ortho_is_thin(rows, cols)) return ortho_thin_bwd(batch, rows, cols, dtype, x, v_y, v_x, co, eps, stream);
    const OrthoPlan p = make_plan(rows, cols, dtype, co, true, kept != nullptr);
    const long long chunk = kept ? batch : ortho_chunk(p, batch);
    for (long long b = 0; b < batch; b += chunk) {
        if (int e = ortho_tiled_bwd(p, co, std::min(chunk, batch - b), at_matrix(x, b, rows, cols, dtype),
                                    at_matrix(v_y, b, rows, cols, dtype),
                                    const_cast<char *>(at_matrix(v_x, b, rows, cols, dtype)), dtype, eps, kept,
                                    static_cast<char *>(scratch), stream))
            return e;
    }
    return kOk;
}

// The matrices [from, from + n) of a table.
static MuonTable table_part(const MuonTable &all, long long from, long long n, int rows, int cols) {
    MuonTable t = all;
    t.n = 0;
    for (int i = 0; i < all.n; ++i) {
        const long long lo = std::max(all.first[i], from), hi = std::min(all.first[i + 1], from + n);
        if (lo >= hi) continue;
        const long long skip = lo - all.first[i];
        t.param[t.n] = const_cast<char *>(at_matrix(all.param[i], skip, rows, cols, all.dtype));
        t.grad[t.n] = at_matrix(all.grad[i], skip, rows, cols, all.dtype);
        t.momentum[t.n] = const_cast<char *>(at_matrix(all.momentum[i], skip, rows, cols, all.state_dtype));
        t.lr[t.n] = all.lr[i];
        t.decay[t.n] = all.decay[i];
        t.inner[t.n] = all.inner[i];
        t.transposed[t.n] = all.transposed[i];
        t.skipped[t.n] = all.skipped[i] + skip;
        t.first[t.n] = lo - from;
        ++t.n;
    }
    t.first[t.n] = n;
    return t;
}

// How a tensor of a Muon step is computed, and what it is computed together with: thin matrices with those
// of their shape, clustered ones with those of their cluster's size, tiled ones with those of their shape or its transpose.
enum MuonKind : int { kMuonThin, kMuonClustered, kMuonTiled };
struct MuonKey {
    int kind, a, b;
    bool operator==(const MuonKey &o) const { return kind == o.kind && a == o.a && b == o.b; }
};
static MuonKey muon_key(const GsbMuonTensor &t) {
    if (ortho_is_thin(t.rows, t.cols)) return {kMuonThin, t.rows, t.cols};
    if (const int blocks = ortho_is_clustered(t.rows, t.cols)) return {kMuonClustered, blocks, 0};
    return {kMuonTiled, std::min(t.rows, t.cols), std::max(t.rows, t.cols)};
}
static bool muon_empty(const GsbMuonTensor &t) { return t.batch == 0 || t.rows == 0 || t.cols == 0; }
// A list is taken in slices, whose keys are worked out once; tensors of different slices are not computed together.
constexpr int kMuonSlice = 256;
struct MuonSlice {
    int n;
    const GsbMuonTensor *tensors;
    MuonKey keys[kMuonSlice];

    MuonSlice(const GsbMuonTensor *all, int from, int count) : n(std::min(count - from, kMuonSlice)), tensors(all + from) {
        for (int i = 0; i < n; ++i) keys[i] = muon_empty(tensors[i]) ? MuonKey{-1, 0, 0} : muon_key(tensors[i]);
    }
    bool leads(int i) const { // whether tensor i is the first of its key
        if (keys[i].kind < 0) return false;
        for (int j = 0; j < i; ++j)
            if (keys[j] == keys[i]) return false;
        return true;
    }
    long long matrices(const MuonKey &key) const {
        long long total = 0;
        for (int i = 0; i < n; ++i)
            if (keys[i] == key) total += tensors[i].batch;
        return total;
    }
};
static int check_tensors(int n_tensors, const GsbMuonTensor *tensors) {
    if (n_tensors < 0) return set_error(kErrInvalidArgument, "muon: negative tensor count");
    if (n_tensors > 0 && tensors == nullptr) return set_error(kErrInvalidArgument, "muon: no tensor list");
    for (int i = 0; i < n_tensors; ++i) {
        const GsbMuonTensor &t = tensors[i];
        if (t.batch < 0 || t.rows < 0 || t.cols < 0 || std::max(t.rows, t.cols) > kOrthoMaxSide || t.inner < 1)
            return set_error(kErrInvalidArgument, "muon: tensor %d: %lld x [%d, %d], inner %d", i, t.batch, t.rows, t.cols, t.inner);
        if (!(t.gain == tensors[0].gain)) return set_error(kErrInvalidArgument, "muon: tensor %d: a gain of its own", i);
    }
    return kOk;
}

extern "C" size_t gsb_muon_scratch_bytes(int n_tensors, const GsbMuonTensor *tensors, int dtype, int steps) {
    if (check_tensors(n_tensors, tensors) != kOk || steps < 1 || steps > kOrthoMaxSteps) return 0;
    OrthoCoefficients co = {};
    co.steps = steps;
    size_t most = 0;
    for (int from = 0; from < n_tensors; from += kMuonSlice) {
        const MuonSlice slice(tensors, from, n_tensors);
        for (int i = 0; i < slice.n; ++i) {
            const MuonKey &key = slice.keys[i];
            if (key.kind == kMuonTiled && slice.leads(i))
                most = std::max(most, plan_bytes(ortho_plan(key.a, key.b, dtype, co, false, false), slice.matrices(key)));
        }
    }
    return most;
}

extern "C" int gsb_muon(int n_tensors, const GsbMuonTensor *tensors, int dtype, int state_dtype, const bool *valid, float momentum,
                        int nesterov, int steps, const float *coefficients, float eps, void *scratch, size_t scratch_bytes,
                        cudaStream_t stream) {
    OrthoCoefficients co = {};
    if (int e = check_common("muon", 0, 0, 0, dtype, steps, coefficients, eps, &co)) return e;
    if (state_dtype != dtype && state_dtype != kOrthoF32)
        return set_error(kErrUnsupported, "muon: the momentum buffer has the parameter's type or float32");
    if (int e = check_tensors(n_tensors, tensors)) return e;
    const size_t needed = gsb_muon_scratch_bytes(n_tensors, tensors, dtype, steps);
    if (needed > 0 && (scratch == nullptr || scratch_bytes < needed))
        return set_error(kErrInvalidArgument, "muon: %zu scratch bytes are needed", needed);
    if (int e = check_room("muon", needed > 0 ? scratch : nullptr)) return e;
    for (int i = 0; i < n_tensors; ++i) {
        const GsbMuonTensor &u = tensors[i];
        if (muon_empty(u)) continue;
        if (int e = check_tensor("muon", u.param, dtype)) return e;
        if (int e = check_tensor("muon", u.grad, dtype)) return e;
        if (int e = check_tensor("muon", u.momentum_buffer, state_dtype)) return e;
    }
    MuonTable t = {};
    t.dtype = dtype;
    t.state_dtype = state_dtype;
    t.nesterov = nesterov;
    const float gain = n_tensors > 0 ? tensors[0].gain : 0.f;
    t.mu = momentum;
    t.one_minus_mu = gain != 0.f ? gain : (float)(1.0 - (double)momentum);
    t.valid = valid;
    int sizes[kOrthoMaxTensors][2]; // rows and columns of the tensors in t
    for (int from = 0; from < n_tensors; from += kMuonSlice) {
        const MuonSlice slice(tensors, from, n_tensors);
        for (int i = 0; i < slice.n; ++i) {
            if (!slice.leads(i)) continue;
            const MuonKey key = slice.keys[i];
            OrthoPlan p = {};
            long long chunk = 0;
            if (key.kind != kMuonThin) p = make_plan(slice.tensors[i].rows, slice.tensors[i].cols, dtype, co, false, false);
            if (key.kind == kMuonTiled) {
                p = make_plan(key.a, key.b, dtype, co, false, false);
                chunk = ortho_chunk(p, slice.matrices(key));
            }
            auto run = [&]() -> int { // the tensors gathered in t
                if (t.n == 0) return kOk;
                int e = kOk;
                if (key.kind == kMuonThin) {
                    e = ortho_thin_muon(t, key.a, key.b, co, eps, stream);
                } else if (key.kind == kMuonClustered) {
                    e = ortho_cluster_muon(t, sizes, co, (float)p.s.x, (float)p.s.a, (float)p.s.b, eps, stream);
                } else {
                    const long long here = t.first[t.n];
                    for (long long b = 0; b < here && e == kOk; b += chunk) {
                        const long long n = std::min(chunk, here - b);
                        e = ortho_tiled_fwd(p, co, n, nullptr, nullptr, dtype, table_part(t, b, n, key.a, key.b), eps,
                                            static_cast<char *>(scratch), stream);
                    }
                }
                t.n = 0;
                return e;
            };
            for (int j = i; j < slice.n; ++j) {
                const GsbMuonTensor &u = slice.tensors[j];
                if (!(slice.keys[j] == key)) continue;
                t.param[t.n] = u.param;
                t.grad[t.n] = u.grad;
                t.momentum[t.n] = u.momentum_buffer;
                t.lr[t.n] = u.lr;
                t.decay[t.n] = u.decay;
                t.inner[t.n] = u.inner;
                t.transposed[t.n] = u.rows > u.cols;
                t.first[t.n + 1] = t.first[t.n] + u.batch;
                sizes[t.n][0] = u.rows;
                sizes[t.n][1] = u.cols;
                if (++t.n == kOrthoMaxTensors)
                    if (int e = run()) return e;
            }
            if (int e = run()) return e;
        }
    }
    return kOk;
}
