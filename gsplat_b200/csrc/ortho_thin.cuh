// Newton-Schulz orthogonalisation of many thin matrices (short side S <= 4, long
// side L <= 128): forward, backward and the whole Muon step, one launch each.
//
// X stays in registers through all steps: the S x S Gram matrix A, its polynomial B, and X (a I + B), one S x S product
// a row, all in 32 bits. Rows past L are zeros, which the iteration leaves zero.
// Memory is read and written once. Two layouts:
//  - "stacked", for many matrices with L <= 32: a thread holds one matrix, two rows to a
//    paired 32-bit instruction, and its block moves the matrices between global and shared memory
//    in their own order. Nothing is repeated or shuffled, which matters since the
//    instruction issue, not memory, bounded the other layout (83% of issue slots
//    and 11% of DRAM at 1M x [15, 3]). 1M x [15, 3] fp32: forward 80 us (4.5 TB/s; 70% of issue slots, 19 warps an SM), Muon
//    step 147 (6.1 TB/s), with 45% of the matrices visible 136 (39% of issue slots, 15 warps), backward 330: every step's X lies in shared
//    memory, which leaves room for 6 warps an SM (44% of issue slots).
//  - "grouped", for few matrices or long ones: 2^g lanes hold one matrix, four rows a
//    lane, and A is summed over them with shuffles.
#pragma once

#include <algorithm>

#include "ortho.cuh"

namespace gsb {

constexpr int kThinRows = 4;
constexpr int kThinThreads = 128;
constexpr int kThinMaxShort = 4;
constexpr int kThinMaxLong = kThinRows * 32;

template <int S> struct Sym { // symmetric S x S, upper triangle by rows
    float v[S * (S + 1) / 2];
    __device__ __forceinline__ static constexpr int at(int i, int j) {
        return (i < j ? i : j) * S - (i < j ? i : j) * ((i < j ? i : j) - 1) / 2 + (i < j ? j - i : i - j);
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

// The Frobenius norm over the group, in 64 bits (any finite input).
template <int S> __device__ __forceinline__ double frobenius(const float x[kThinRows][S], int group) {
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) s = fma((double)x[r][j], (double)x[r][j], s);
    return sqrt(group_sum(s, group));
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
    thin_fwd_kernel(ThinShape sh, const T *__restrict__ x_in, T *__restrict__ y, const __grid_constant__ OrthoCoefficients co, float eps) {
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
    const Divisor d = divisor_of(frobenius<S>(x, sh.group), eps);
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] * d.pre / d.div;
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
                    const __grid_constant__ OrthoCoefficients co, float eps) {
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
    const Divisor d = divisor_of(frobenius<S>(x, sh.group), eps);
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] * d.pre / d.div;
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
    if (d.small) dot = 0.f;
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int l = r * sh.group + lane;
            if (live && l < sh.L)
                v_x[base + l * sh.row_step + j * sh.col_step] = from_f32<T>(fmaf(-x[r][j], dot, g[r][j]) / d.div * d.pre);
        }
}

// Momentum, orthogonalisation and the parameters' step in one pass. Matrices of
// hidden rows keep their values.
template <typename T, typename M, int S>
__global__ void __launch_bounds__(kThinThreads)
    thin_muon_kernel(ThinShape sh, const __grid_constant__ MuonTable tab, const __grid_constant__ OrthoCoefficients co, float eps) {
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
    const Divisor d = divisor_of(frobenius<S>(x, sh.group), eps);
#pragma unroll
    for (int r = 0; r < kThinRows; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = x[r][j] * d.pre / d.div;
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

// --- stacked -------------------------------------------------------------------
constexpr int kStackThreads = 128;
constexpr int kStackMaxLong = 32;
constexpr int kStackMaxLongBwd = 16; // X and G of 32 rows do not fit the registers

__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 halves(uint64_t a) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(a));
    return v;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

template <int P, int S> __device__ __forceinline__ Sym<S> pair_gram(const uint64_t x[P][S]) {
    Sym<S> a;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = i; j < S; ++j) {
            uint64_t s = pair_mul(x[0][i], x[0][j]);
#pragma unroll
            for (int r = 1; r < P; ++r) s = pair_fma(x[r][i], x[r][j], s);
            const float2 h = halves(s);
            a(i, j) = h.x + h.y;
        }
    return a;
}
template <int P, int S>
__device__ __forceinline__ Sym<S> pair_cross(const uint64_t x[P][S], const uint64_t y[P][S]) {
    Sym<S> a;
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = i; j < S; ++j) {
            uint64_t s = 0;
#pragma unroll
            for (int r = 0; r < P; ++r) s = pair_fma(x[r][i], y[r][j], pair_fma(y[r][i], x[r][j], s));
            const float2 h = halves(s);
            a(i, j) = h.x + h.y;
        }
    return a;
}
// y <- x (a I + B), or y + x B
template <int P, int S, bool ADD>
__device__ __forceinline__ void pair_apply(const uint64_t x[P][S], uint64_t y[P][S], const Sym<S> &B, float a) {
    uint64_t m[S][S];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const float v = i == j && !ADD ? a + B(i, i) : B(i, j);
            m[i][j] = pair_of(v, v);
        }
#pragma unroll
    for (int r = 0; r < P; ++r) {
        uint64_t t[S];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            t[j] = ADD ? pair_fma(x[r][0], m[0][j], y[r][j]) : pair_mul(x[r][0], m[0][j]);
#pragma unroll
            for (int k = 1; k < S; ++k) t[j] = pair_fma(x[r][k], m[k][j], t[j]);
        }
#pragma unroll
        for (int j = 0; j < S; ++j) y[r][j] = t[j];
    }
}

// X <- X / max(|X|, eps). The sum of squares is of values brought near 1 by a power of
// two, so neither overflows nor vanishes. Returns what a value of X was multiplied with:
// first by `scale`, then by `inv`; `small`: the norm was below eps.
struct ThinNorm {
    float scale, inv;
    bool small;
};
template <int P, int S> __device__ __forceinline__ ThinNorm pair_normalize(uint64_t x[P][S], float eps) {
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < P; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const float2 h = halves(x[r][j]);
            top = fmaxf(top, fmaxf(fabsf(h.x), fabsf(h.y)));
        }
    ThinNorm n;
    const int e = __float_as_int(top) >> 23; // 255: infinite; a NaN is not seen here, but in the sum
    n.scale = e == 255 || top == 0.f ? 1.f : __int_as_float(max(1, 254 - e) << 23);
    const uint64_t sc = pair_of(n.scale, n.scale);
    uint64_t s = 0;
#pragma unroll
    for (int r = 0; r < P; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            x[r][j] = pair_mul(x[r][j], sc);
            s = pair_fma(x[r][j], x[r][j], s);
        }
    const float2 h = halves(s);
    const float norm = sqrtf(h.x + h.y);
    n.small = norm < eps * n.scale;
    // eps may be far above the values: its scaled form may overflow, and 1 / it vanish, as X does
    n.inv = n.small ? 1.f / (eps * n.scale) : 1.f / norm;
    const uint64_t iv = pair_of(n.inv, n.inv);
#pragma unroll
    for (int r = 0; r < P; ++r)
#pragma unroll
        for (int j = 0; j < S; ++j) x[r][j] = pair_mul(x[r][j], iv);
    return n;
}

struct StackShape {
    long long batch;
    int L, E, pitch; // rows, values of a matrix, floats between two in shared memory (odd: no two threads on a bank)
    int tall; // stored [L, S], else [S, L]
    int vec;  // the tensors may be read four values at a time
    uint32_t magic; // ceil(2^32 / E): value e < 2^16 belongs to matrix (e magic) >> 32
    uint32_t magic_quads; // and of the quads a matrix can touch, (E + 6) / 4
};

// Row l of 2 P: rows below P are always there (P is the smallest that holds L), save for the least P.
template <int P> __device__ __forceinline__ bool stack_row(const StackShape &sh, int l) {
    return (P > 2 && l < P) || l < sh.L;
}
template <int P, int S, bool TALL>
__device__ __forceinline__ void stack_read_as(const StackShape &sh, const float *own, uint64_t x[P][S]) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const float *col = TALL ? own + j : own + j * sh.L;
        constexpr int step = TALL ? S : 1;
#pragma unroll
        for (int r = 0; r < P; ++r)
            x[r][j] = pair_of(stack_row<P>(sh, 2 * r) ? col[2 * r * step] : 0.f,
                              stack_row<P>(sh, 2 * r + 1) ? col[(2 * r + 1) * step] : 0.f);
    }
}
template <int P, int S>
__device__ __forceinline__ void stack_read(const StackShape &sh, const float *own, uint64_t x[P][S]) {
    if (sh.tall) stack_read_as<P, S, true>(sh, own, x);
    else stack_read_as<P, S, false>(sh, own, x);
}
template <int P, int S, bool TALL>
__device__ __forceinline__ void stack_write_as(const StackShape &sh, float *own, const uint64_t x[P][S]) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
        float *col = TALL ? own + j : own + j * sh.L;
        constexpr int step = TALL ? S : 1;
#pragma unroll
        for (int r = 0; r < P; ++r) {
            const float2 h = halves(x[r][j]);
            if (stack_row<P>(sh, 2 * r)) col[2 * r * step] = h.x;
            if (stack_row<P>(sh, 2 * r + 1)) col[(2 * r + 1) * step] = h.y;
        }
    }
}
template <int P, int S>
__device__ __forceinline__ void stack_write(const StackShape &sh, float *own, const uint64_t x[P][S]) {
    if (sh.tall) stack_write_as<P, S, true>(sh, own, x);
    else stack_write_as<P, S, false>(sh, own, x);
}
__device__ __forceinline__ int stack_matrix(const StackShape &sh, int e) {
    return sh.E == 1 ? e : (int)__umulhi((uint32_t)e, sh.magic);
}

// Quad i of the stage. With an odd E the stage lies as memory does; else a matrix
// is followed by one float of padding, which a quad may straddle (E >= 4).
__device__ __forceinline__ void stage_put(const StackShape &sh, float *stage, int i, float4 f) {
    if (sh.pitch == sh.E) {
        reinterpret_cast<float4 *>(stage)[i] = f;
    } else {
        const int q = stack_matrix(sh, 4 * i), left = (q + 1) * sh.E - 4 * i; // values until the padding
        float *at = stage + 4 * i + q;
        at[0] = f.x;
        at[left > 1 ? 1 : 2] = f.y;
        at[left > 2 ? 2 : 3] = f.z;
        at[left > 3 ? 3 : 4] = f.w;
    }
}
__device__ __forceinline__ float4 stage_get(const StackShape &sh, const float *stage, int i) {
    if (sh.pitch == sh.E) return reinterpret_cast<const float4 *>(stage)[i];
    const int q = stack_matrix(sh, 4 * i), left = (q + 1) * sh.E - 4 * i;
    const float *at = stage + 4 * i + q;
    return make_float4(at[0], at[left > 1 ? 1 : 2], at[left > 2 ? 2 : 3], at[left > 3 ? 3 : 4]);
}

// The block's n matrices from `in` to the stage, or from the stage to `out`. A block's first value
// is at a multiple of 64 E, so four at a time are aligned where the
// tensor is; several are on their way at once, since nothing else hides the latency.
template <typename T>
__device__ __forceinline__ void stack_load(const StackShape &sh, const T *__restrict__ in, int n, float *stage) {
    const int total = n * sh.E, quads = sh.vec ? total / 4 : 0;
    using V = typename Quad<T>::type;
    constexpr int U = 8;
    for (int i0 = threadIdx.x; i0 < quads; i0 += U * blockDim.x) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * blockDim.x < quads) v[u] = reinterpret_cast<const V *>(in)[i0 + u * blockDim.x];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * blockDim.x < quads) stage_put(sh, stage, i0 + u * blockDim.x, Quad<T>::get(v[u]));
    }
#pragma unroll 4
    for (int e = 4 * quads + threadIdx.x; e < total; e += blockDim.x) {
        const int q = stack_matrix(sh, e);
        stage[q * sh.pitch + e - q * sh.E] = to_f32(in[e]);
    }
}
template <typename T>
__device__ __forceinline__ void stack_store(const StackShape &sh, const float *stage, int n, T *__restrict__ out) {
    const int total = n * sh.E, quads = sh.vec ? total / 4 : 0;
    using V = typename Quad<T>::type;
#pragma unroll 4
    for (int i = threadIdx.x; i < quads; i += blockDim.x)
        reinterpret_cast<V *>(out)[i] = Quad<T>::put(stage_get(sh, stage, i));
#pragma unroll 4
    for (int e = 4 * quads + threadIdx.x; e < total; e += blockDim.x) {
        const int q = stack_matrix(sh, e);
        out[e] = from_f32<T>(stage[q * sh.pitch + e - q * sh.E]);
    }
}

template <int P, int S>
__device__ __forceinline__ void pair_iterate(uint64_t x[P][S], const OrthoCoefficients &co) {
    for (int k = 0; k < co.steps; ++k)
        pair_apply<P, S, false>(x, x, poly<S>(pair_gram<P, S>(x), co.c[k][1], co.c[k][2]), co.c[k][0]);
}

template <typename T, int P, int S>
__global__ void __launch_bounds__(kStackThreads)
    stack_fwd_kernel(StackShape sh, const T *__restrict__ x_in, T *__restrict__ y, const __grid_constant__ OrthoCoefficients co, float eps) {
    extern __shared__ __align__(16) float stage[];
    const long long b0 = (long long)blockIdx.x * kStackThreads;
    const int n = (int)min((long long)kStackThreads, sh.batch - b0);
    const size_t base = (size_t)b0 * sh.E;
    stack_load(sh, x_in + base, n, stage);
    __syncthreads();
    if ((int)threadIdx.x < n) {
        float *own = stage + threadIdx.x * sh.pitch;
        uint64_t x[P][S];
        stack_read<P, S>(sh, own, x);
        pair_normalize<P, S>(x, eps);
        pair_iterate<P, S>(x, co);
        stack_write<P, S>(sh, own, x);
    }
    __syncthreads();
    stack_store(sh, stage, n, y + base);
}

// Every step's X is kept in shared memory behind the stage, [step][value][thread].
template <typename T, int P, int S>
__global__ void __launch_bounds__(kStackThreads)
    stack_bwd_kernel(StackShape sh, const T *__restrict__ x_in, const T *__restrict__ v_y, T *__restrict__ v_x,
                     const __grid_constant__ OrthoCoefficients co, float eps) {
    extern __shared__ __align__(16) float stage[];
    const int threads = blockDim.x;
    uint64_t *kept = reinterpret_cast<uint64_t *>(stage + ((threads * sh.pitch + 1) & ~1)) + threadIdx.x;
    const long long b0 = (long long)blockIdx.x * threads;
    const int n = (int)min((long long)threads, sh.batch - b0);
    const size_t base = (size_t)b0 * sh.E;
    float *own = stage + threadIdx.x * sh.pitch;
    const bool live = (int)threadIdx.x < n;
    stack_load(sh, x_in + base, n, stage);
    __syncthreads();
    uint64_t x[P][S], g[P][S];
    if (live) stack_read<P, S>(sh, own, x);
    __syncthreads();
    stack_load(sh, v_y + base, n, stage);
    __syncthreads();
    if (live) {
        stack_read<P, S>(sh, own, g);
        const ThinNorm norm = pair_normalize<P, S>(x, eps);
        for (int k = 0; k < co.steps; ++k) {
#pragma unroll
            for (int r = 0; r < P; ++r)
#pragma unroll
                for (int j = 0; j < S; ++j) kept[((k * P + r) * S + j) * threads] = x[r][j];
            if (k + 1 < co.steps)
                pair_apply<P, S, false>(x, x, poly<S>(pair_gram<P, S>(x), co.c[k][1], co.c[k][2]), co.c[k][0]);
        }
        for (int k = co.steps - 1; k >= 0; --k) {
            const float cb = co.c[k][1], cc = co.c[k][2];
#pragma unroll
            for (int r = 0; r < P; ++r)
#pragma unroll
                for (int j = 0; j < S; ++j) x[r][j] = kept[((k * P + r) * S + j) * threads];
            const Sym<S> A = pair_gram<P, S>(x), Q = pair_cross<P, S>(x, g);
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
            pair_apply<P, S, false>(g, g, poly<S>(A, cb, cc), co.c[k][0]);
            pair_apply<P, S, true>(x, g, t, 0.f);
        }
        // x holds X0: dU = (G - X0 <G, X0>) / |U|, or G / eps below eps
        uint64_t d = 0;
#pragma unroll
        for (int r = 0; r < P; ++r)
#pragma unroll
            for (int j = 0; j < S; ++j) d = pair_fma(g[r][j], x[r][j], d);
        const float2 h = halves(d);
        const float dot = norm.small ? 0.f : -(h.x + h.y);
        const float inv = norm.small ? 1.f / eps : norm.inv, scale = norm.small ? 1.f : norm.scale;
        const uint64_t dd = pair_of(dot, dot), sc = pair_of(scale, scale), iv = pair_of(inv, inv);
#pragma unroll
        for (int r = 0; r < P; ++r)
#pragma unroll
            for (int j = 0; j < S; ++j) g[r][j] = pair_mul(pair_mul(pair_fma(x[r][j], dd, g[r][j]), iv), sc);
        stack_write<P, S>(sh, own, g);
    }
    __syncthreads();
    stack_store(sh, stage, n, v_x + base);
}

// The Muon step. A block takes `span` consecutive matrices of one tensor: it moves the visible ones as
// they lie in memory, four values at a time, and lists them, so that its threads take
// them kStackThreads at a time and a mask leaves few of them idle.
constexpr int kStackSpan = 4 * kStackThreads; // at most

struct StackBlocks {
    long long first[kOrthoMaxTensors + 1]; // the first block of each tensor
    int vec[kOrthoMaxTensors];             // the tensor may be moved four values at a time
    int span;
};

template <typename T, typename M, int P, int S>
__global__ void __launch_bounds__(kStackThreads)
    stack_muon_kernel(StackShape sh, const __grid_constant__ MuonTable tab, const __grid_constant__ StackBlocks blocks,
                      const __grid_constant__ OrthoCoefficients co, float eps) {
    extern __shared__ __align__(16) float stage[];
    __shared__ short list[kStackSpan];
    __shared__ bool visible[kStackSpan + 1];
    __shared__ int warp_count[kStackThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int t = 0;
    while (t + 1 < tab.n && (long long)blockIdx.x >= blocks.first[t + 1]) ++t;
    const long long in_tensor = ((long long)blockIdx.x - blocks.first[t]) * blocks.span;
    const int n = (int)min((long long)blocks.span, tab.first[t + 1] - tab.first[t] - in_tensor);
    int count = 0;
    for (int i = 0; i < n; i += kStackThreads) {
        const int q = i + threadIdx.x;
        const bool seen = q < n && muon_visible(tab, t, tab.first[t] + in_tensor + q);
        const unsigned mask = __ballot_sync(0xffffffffu, seen);
        if (lane == 0) warp_count[warp] = __popc(mask);
        if (q < n) visible[q] = seen;
        __syncthreads();
        int before = count;
#pragma unroll
        for (int w = 0; w < kStackThreads / 32; ++w) {
            if (w < warp) before += warp_count[w];
            count += warp_count[w];
        }
        if (seen) list[before + __popc(mask & ((1u << lane) - 1))] = (short)q;
        __syncthreads();
    }
    if (count == 0) return;
    const bool all = count == n;
    const size_t base = (size_t)in_tensor * sh.E;
    const T *grad = static_cast<const T *>(tab.grad[t]) + base;
    M *mom = static_cast<M *>(tab.momentum[t]) + base;
    T *param = static_cast<T *>(tab.param[t]) + base;
    const int total = n * sh.E;
    auto one_in = [&](int e) {
        const int q = stack_matrix(sh, e);
        if (!visible[q]) return;
        const float g = to_f32(grad[e]), m = muon_momentum(g, to_f32(mom[e]), tab.one_minus_mu);
        mom[e] = from_f32<M>(m);
        stage[q * sh.pitch + e - q * sh.E] = muon_update(g, m, tab.mu, tab.nesterov);
    };
    auto one_out = [&](int e) {
        const int q = stack_matrix(sh, e);
        if (!visible[q]) return;
        param[e] = from_f32<T>(muon_param(to_f32(param[e]), stage[q * sh.pitch + e - q * sh.E], tab.lr[t], tab.decay[t]));
    };
    using VT = typename Quad<T>::type;
    using VM = typename Quad<M>::type;
    constexpr int U = 4; // quads on their way at once
    auto updated = [&](float4 g, float4 &m) -> float4 {
        m = make_float4(muon_momentum(g.x, m.x, tab.one_minus_mu), muon_momentum(g.y, m.y, tab.one_minus_mu),
                        muon_momentum(g.z, m.z, tab.one_minus_mu), muon_momentum(g.w, m.w, tab.one_minus_mu));
        return make_float4(muon_update(g.x, m.x, tab.mu, tab.nesterov), muon_update(g.y, m.y, tab.mu, tab.nesterov),
                           muon_update(g.z, m.z, tab.mu, tab.nesterov), muon_update(g.w, m.w, tab.mu, tab.nesterov));
    };
    // With hidden matrices, each listed one's quads in turn (turn `at` of `turns`): quad i, the values of it that are the
    // matrix's, and their place on the stage. A quad that it shares is read whole and written value by value.
    const int per = (sh.E + 6) / 4, turns = !blocks.vec[t] || all ? 0 : count * per, quads = blocks.vec[t] && all ? total / 4 : 0;
    struct Part {
        int i;
        unsigned seen;
        float *stage;
    };
    auto part = [&](int at) -> Part {
        const int l = (int)__umulhi((uint32_t)at, sh.magic_quads), q = list[l], first = q * sh.E, i = first / 4 + at - l * per;
        const int from = first - 4 * i, to = first + sh.E - 4 * i; // of the quad, 0 to 4
        return {i, to <= 0 ? 0u : (15u >> max(0, 4 - to)) & (15u << max(0, from)), stage + 4 * i + (sh.pitch != sh.E ? q : 0)};
    };
    for (int i0 = threadIdx.x; i0 < quads; i0 += U * kStackThreads) {
        float4 g[U], m[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * kStackThreads < quads) {
                g[u] = Quad<T>::get(reinterpret_cast<const VT *>(grad)[i0 + u * kStackThreads]);
                m[u] = Quad<M>::get(reinterpret_cast<const VM *>(mom)[i0 + u * kStackThreads]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * kStackThreads < quads) {
                const float4 w = updated(g[u], m[u]);
                reinterpret_cast<VM *>(mom)[i0 + u * kStackThreads] = Quad<M>::put(m[u]);
                stage_put(sh, stage, i0 + u * kStackThreads, w);
            }
    }
    for (int a0 = threadIdx.x; a0 < turns; a0 += U * kStackThreads) {
        float4 g[U], m[U];
        Part at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = a0 + u * kStackThreads < turns ? part(a0 + u * kStackThreads) : Part{0, 0u, stage};
            if (at[u].seen && 4 * at[u].i + 3 < total) {
                g[u] = Quad<T>::get(reinterpret_cast<const VT *>(grad)[at[u].i]);
                m[u] = Quad<M>::get(reinterpret_cast<const VM *>(mom)[at[u].i]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned seen = at[u].seen;
            if (!seen) continue;
            if (4 * at[u].i + 3 >= total) { // the tensor's last values
#pragma unroll 1
                for (int e = 4 * at[u].i; e < total; ++e) one_in(e);
                continue;
            }
            const float4 w = updated(g[u], m[u]);
            float *own = at[u].stage;
            M *to = mom + 4 * at[u].i;
            if (seen & 1u) own[0] = w.x;
            if (seen & 2u) own[1] = w.y;
            if (seen & 4u) own[2] = w.z;
            if (seen & 8u) own[3] = w.w;
            if (seen == 15u) {
                *reinterpret_cast<VM *>(to) = Quad<M>::put(m[u]);
            } else {
                if (seen & 1u) to[0] = from_f32<M>(m[u].x);
                if (seen & 2u) to[1] = from_f32<M>(m[u].y);
                if (seen & 4u) to[2] = from_f32<M>(m[u].z);
                if (seen & 8u) to[3] = from_f32<M>(m[u].w);
            }
        }
    }
    for (int e = (!blocks.vec[t] ? 0 : all ? 4 * quads : total) + threadIdx.x; e < total; e += kStackThreads) one_in(e);
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kStackThreads) {
        float *own = stage + list[i] * sh.pitch;
        uint64_t x[P][S];
        stack_read<P, S>(sh, own, x);
        pair_normalize<P, S>(x, eps);
        pair_iterate<P, S>(x, co);
        stack_write<P, S>(sh, own, x);
    }
    __syncthreads();
    const float lr = tab.lr[t], decay = tab.decay[t];
    for (int i0 = threadIdx.x; i0 < quads; i0 += U * kStackThreads) {
        float4 p[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * kStackThreads < quads) p[u] = Quad<T>::get(reinterpret_cast<const VT *>(param)[i0 + u * kStackThreads]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * kStackThreads < quads) {
                const float4 o = stage_get(sh, stage, i0 + u * kStackThreads);
                reinterpret_cast<VT *>(param)[i0 + u * kStackThreads] =
                    Quad<T>::put(make_float4(muon_param(p[u].x, o.x, lr, decay), muon_param(p[u].y, o.y, lr, decay),
                                             muon_param(p[u].z, o.z, lr, decay), muon_param(p[u].w, o.w, lr, decay)));
            }
    }
    for (int a0 = threadIdx.x; a0 < turns; a0 += U * kStackThreads) {
        float4 p[U];
        Part at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = a0 + u * kStackThreads < turns ? part(a0 + u * kStackThreads) : Part{0, 0u, stage};
            if (at[u].seen && 4 * at[u].i + 3 < total) p[u] = Quad<T>::get(reinterpret_cast<const VT *>(param)[at[u].i]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned seen = at[u].seen;
            if (!seen) continue;
            if (4 * at[u].i + 3 >= total) {
#pragma unroll 1
                for (int e = 4 * at[u].i; e < total; ++e) one_out(e);
                continue;
            }
            // beside the matrix's values lie others, or the room behind the stage, which are not used
            const float *own = at[u].stage;
            T *to = param + 4 * at[u].i;
            const float4 w = make_float4(muon_param(p[u].x, own[0], lr, decay), muon_param(p[u].y, own[1], lr, decay),
                                         muon_param(p[u].z, own[2], lr, decay), muon_param(p[u].w, own[3], lr, decay));
            if (seen == 15u) {
                *reinterpret_cast<VT *>(to) = Quad<T>::put(w);
            } else {
                if (seen & 1u) to[0] = from_f32<T>(w.x);
                if (seen & 2u) to[1] = from_f32<T>(w.y);
                if (seen & 4u) to[2] = from_f32<T>(w.z);
                if (seen & 8u) to[3] = from_f32<T>(w.w);
            }
        }
    }
    for (int e = (!blocks.vec[t] ? 0 : all ? 4 * quads : total) + threadIdx.x; e < total; e += kStackThreads) one_out(e);
}

inline ThinShape thin_shape(long long batch, int rows, int cols) {
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
inline unsigned thin_blocks(const ThinShape &sh, int threads) {
    const int per_block = threads / sh.group;
    const long long n = (sh.batch + per_block - 1) / per_block;
    return n > 0x7fffffffll ? 0u : (unsigned)n;
}

template <typename F> inline int with_short(int S, F f) {
    switch (S) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    default: return f(std::integral_constant<int, 4>());
    }
}
inline StackShape stack_shape(long long batch, int rows, int cols) {
    StackShape sh;
    sh.batch = batch;
    sh.L = std::max(rows, cols);
    sh.E = rows * cols;
    sh.pitch = sh.E | 1;
    sh.vec = 0;
    sh.tall = rows >= cols;
    sh.magic_quads = ~0u / (uint32_t)((sh.E + 6) / 4) + 1u;
    sh.magic = sh.E <= 1 ? 0u : ~0u / (uint32_t)sh.E + 1u;
    return sh;
}

inline bool quads_aligned(const void *p, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % (dtype == kOrthoF32 ? 16 : 8) == 0;
}
constexpr int kStackSmem = 100 * 1024; // two blocks an SM

// f with the row pairs P (rows rounded up) and S as constants
template <int MOST, typename F> inline int with_rows(int L, F f) {
    if (L <= 4) return f(std::integral_constant<int, 2>());
    if (L <= 8) return f(std::integral_constant<int, 4>());
    if (MOST == 16 || L <= 16) return f(std::integral_constant<int, 8>());
    return f(std::integral_constant<int, MOST / 2>());
}
template <typename K> inline bool allow_smem(K kernel, size_t smem) {
    return smem <= 40 * 1024 || // with the kernels' own few KiB below the 48 that need no permission
           cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
}

template <typename F> inline int with_type(int dtype, F f) {
    if (dtype == kOrthoF32) return f(float());
    if (dtype == kOrthoBF16) return f(__nv_bfloat16());
    return f(__half());
}

} // namespace gsb
