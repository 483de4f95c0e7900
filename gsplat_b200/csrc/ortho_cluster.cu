// Newton-Schulz steps of matrices whose short side is at most 128, in one launch: a
// cluster of blocks holds a matrix X [m, n] in shared memory, each block a slab of its columns, from
// the first read to the last write.
//
// What bounds such a matrix is not its products but the chain of them: 15 launches of
// the tiled kernel took 165 us for a stack of 64 x 64, this takes 25 ([77, 1000] x 12 54, [128, 1024] 69; a step of 64 x 64 3.8,
// a third each for A, B and X: 0.7 until the product is there, 0.4 for its end). Here a step is
//   A = X X^T      each block multiplies its slab; with several blocks the partial
//                  sums are exchanged through distributed shared memory (each block adds up some rows
//                  of A, in the order of the blocks, and gives them to all)
//   B = b A + c A A  every block for itself: m x m is little work, and nothing need be sent
//   X <- a X + B X   each block its slab
// with tcgen05.mma from 128-byte-swizzled planes that serve as depth-major operand of X X^T
// and as column-major operand of B X alike. X, A and B are pairs of fp16 planes (hi, lo) and
// every product is the sum hi hi + hi lo + lo hi; A and B share their place, and the
// diagonals stay in 32 bits, as orthogonalize.cu describes. A thread owns row i of the accumulator and takes 16 columns at a time,
// the four warps of a lane quarter taking turns.
#include <algorithm>

#include "ortho.cuh"
#include "tcgen05.cuh"

namespace gsb {

constexpr int kClusterThreads = 512;
constexpr int kClusterMaxShort = 128;
constexpr int kClusterMax = 8;              // blocks a cluster, the portable limit
constexpr size_t kClusterSmem = 227 * 1024; // of an SM, and a block at most
constexpr size_t kClusterStatic = 4096;     // of which the kernel's own arrays take less than this

struct ClusterShape {
    int m, n, transposed;   // short, long; the tensor is [n, m]
    int m16, mk, ns, ns64;  // rounded up: m to 16 and 64, a block's columns to 16 and 64
    int blocks, columns;    // of a cluster; of TMEM
    int per;                // rows of A that a block of a cluster adds up
    float x_scale, to_a, to_d, unscale_b, unscale_x;
    size_t smem;
};

// The constants of a step: X <- a X + B X; B = c0 .. of A as kEpiSquare of OrthoGemm has it.
struct ClusterSteps {
    int n;
    float c[kOrthoMaxSteps][7]; // a, c0, c1, c2, c3, c4, c5
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ double remote_load_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store4(uint32_t addr, uint4 v) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void remote_store_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// Shared memory written by threads is read by the tensor cores after this and a barrier.
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Byte of (row, column) in a plane of `rows` rows: blocks of 64 columns, rows of 128 bytes
// whose 16-byte pieces are permuted by the row.
__device__ __forceinline__ uint32_t plane_byte(int rows, int row, int col) {
    return (uint32_t)((col >> 6) * rows * 128 + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4) + (col & 7) * 2);
}

__device__ __forceinline__ void split8(const float *v, uint4 &hi, uint4 &lo) {
    __half2 *h = reinterpret_cast<__half2 *>(&hi), *l = reinterpret_cast<__half2 *>(&lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(h[i]);
        l[i] = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    }
}
__device__ __forceinline__ void join8(uint4 hi, uint4 lo, float *v) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&hi), *l = reinterpret_cast<const __half2 *>(&lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(h[i]), b = __half22float2(l[i]);
        v[2 * i] = a.x + b.x;
        v[2 * i + 1] = a.y + b.y;
    }
}
__device__ __forceinline__ void planes_get16(const char *hi, const char *lo, int rows, int row, int col, float v[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = plane_byte(rows, row, col + 8 * h);
        join8(*reinterpret_cast<const uint4 *>(hi + at), *reinterpret_cast<const uint4 *>(lo + at), v + 8 * h);
    }
}
__device__ __forceinline__ void planes_put16(char *hi, char *lo, int rows, int row, int col, const float v[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = plane_byte(rows, row, col + 8 * h);
        uint4 a, b;
        split8(v + 8 * h, a, b);
        *reinterpret_cast<uint4 *>(hi + at) = a;
        *reinterpret_cast<uint4 *>(lo + at) = b;
    }
}

// The descriptors of a product of planes and what a step of 64 of its depth adds to them, in 16-byte units: P
// depth-major; Q depth-major from its first row (X X^T, A A), or column-major (B X). `rows`: of the planes.
struct Operands {
    uint64_t p, p_lo, q, q_lo;
    uint32_t p_block, q_block, q_step; // of 64 deep, and of 16 within
};
__device__ __forceinline__ Operands operands(uint32_t p, uint32_t p_lo, uint32_t q, uint32_t q_lo, int rows, bool q_k_major) {
    const uint32_t chunk = rows * 128;
    return {operand_desc(p, true, 0), operand_desc(p_lo, true, 0), operand_desc(q, q_k_major, chunk), operand_desc(q_lo, q_k_major, chunk),
            chunk / 16, q_k_major ? chunk / 16 : 64 * 128 / 16, q_k_major ? 2u : 128u};
}
// One warp: D[128, n] = P Q over `depth` (a multiple of 16). The small products (hi lo and lo hi) come first: the
// accumulator truncates at every addition, relative to the sum so far, and so only a third of the
// additions are to a large one.
__device__ __forceinline__ void multiply(uint32_t d, const Operands &o, uint32_t idesc, int depth, uint32_t leader) {
    Operands at = o;
    for (int k = 0; k < depth; k += 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + 16 * i >= depth) break;
            mma_f16(d, at.p + 2 * i, at.q_lo + i * o.q_step, idesc, k > 0 || i > 0, leader);
            mma_f16(d, at.p_lo + 2 * i, at.q + i * o.q_step, idesc, true, leader);
        }
        at.p += o.p_block, at.p_lo += o.p_block;
        at.q += o.q_block, at.q_lo += o.q_block;
    }
    at = o;
    for (int k = 0; k < depth; k += 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + 16 * i >= depth) break;
            mma_f16(d, at.p + 2 * i, at.q + i * o.q_step, idesc, true, leader);
        }
        at.p += o.p_block;
        at.q += o.q_block;
    }
}

// The shapes of a launch's tensors; all have the same number of blocks a cluster.
template <bool MUON> struct ClusterShapes {
    ClusterShape of[MUON ? kOrthoMaxTensors : 1];
};

template <typename T, typename M, bool MUON>
__global__ void __launch_bounds__(kClusterThreads, 1)
    ortho_cluster_kernel(const __grid_constant__ ClusterShapes<MUON> shapes, const T *x_in, T *y, const __grid_constant__ MuonTable tab,
                         const __grid_constant__ ClusterSteps co, float eps, const __grid_constant__ ClusterKept kept) {
    extern __shared__ char raw[];
    __shared__ alignas(16) float diag_a[kClusterMaxShort];
    __shared__ float diag_b[kClusterMaxShort];
    __shared__ double warp_sum[kClusterThreads / 32], block_total;
    __shared__ alignas(8) unsigned long long done;
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid % 32;
    const int blocks = shapes.of[0].blocks;
    const uint32_t rank = blocks > 1 ? cluster_rank() : 0;
    const long long b = blockIdx.x / blocks;
    const int tensor = MUON ? muon_tensor_of(tab, b) : 0;
    const ClusterShape &sh = shapes.of[tensor];
    if (MUON && !muon_visible(tab, tensor, b)) return; // the whole cluster alike

    char *base = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int x_plane = sh.m16 * sh.ns64 * 2, a_plane = sh.m16 * sh.mk * 2;
    char *x_hi = base, *x_lo = x_hi + x_plane, *a_hi = x_lo + x_plane, *a_lo = a_hi + a_plane;
    float *partial = reinterpret_cast<float *>(a_lo + a_plane); // several blocks: [blocks][m16 / 4][per], four columns each
    volatile int *abort = &abort_flag;

    const int j0 = (int)rank * sh.ns, cols = max(0, min(sh.ns, sh.n - j0)); // this block's columns
    const size_t numel = (size_t)sh.m * sh.n;
    const size_t mat = (size_t)(MUON ? b - tab.first[tensor] : b) * numel;
    const T *grad = MUON ? static_cast<const T *>(tab.grad[tensor]) + mat : x_in + mat;
    M *mom = MUON ? static_cast<M *>(tab.momentum[tensor]) + mat : nullptr;
    // The slab is moved four values at a time where they lie together and are aligned. Move e of `moves`: its
    // place in the tensor, the row and column of its first value here; with a transposed tensor the next values are
    // further rows, at the last of which the next column begins.
    const int inner = sh.transposed ? sh.m : cols, count = sh.m * cols;
    const uint32_t magic = inner > 1 ? 0xffffffffu / (uint32_t)inner + 1u : 0u;
    const bool whole = sh.transposed || cols == sh.n; // the slab lies in one piece
    bool quads = (whole || (sh.n % 4 == 0 && cols % 4 == 0)) && (whole ? (size_t)j0 * sh.m % 4 == 0 : true);
    if (MUON) {
        T *p = static_cast<T *>(tab.param[tensor]) + mat;
        quads = quads && reinterpret_cast<uintptr_t>(grad) % (4 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 &&
                reinterpret_cast<uintptr_t>(mom) % (4 * sizeof(M)) == 0;
    } else {
        quads = quads && reinterpret_cast<uintptr_t>(grad) % (4 * sizeof(T)) == 0 &&
                reinterpret_cast<uintptr_t>(y + mat) % (4 * sizeof(T)) == 0;
    }
    const int fours = quads ? count / 4 : 0, moves = fours + (count - 4 * fours);
    auto place = [&](int e, int &i, int &j) -> size_t {
        const int v = e < fours ? 4 * e : e + 3 * fours;
        const int o = inner > 1 ? (int)__umulhi((uint32_t)v, magic) : v, k = v - o * inner;
        i = sh.transposed ? k : o;
        j = sh.transposed ? o : k;
        return sh.transposed ? (size_t)j0 * sh.m + v : (size_t)o * sh.n + j0 + k;
    };
    auto next = [&](int &i, int &j) {
        if (sh.transposed) {
            if (++i == sh.m) i = 0, ++j;
        } else if (++j == cols) { // only where the slab is whole rows
            j = 0, ++i;
        }
    };
    using VT = typename Quad<T>::type;
    using VM = typename Quad<M>::type;
    // The matrix to orthogonalise at a move: one value in .x, or four.
    auto fetch = [&](size_t at, bool four, float4 &m) -> float4 {
        float4 g = {};
        m = g;
        if (four) {
            g = Quad<T>::get(*reinterpret_cast<const VT *>(grad + at));
            if (MUON) m = Quad<M>::get(*reinterpret_cast<const VM *>(mom + at));
        } else {
            g.x = to_f32(grad[at]);
            if (MUON) m.x = to_f32(mom[at]);
        }
        return g;
    };
    auto updated = [&](float4 g, float4 &m) -> float4 {
        if (!MUON) return g;
        m.x = muon_momentum(g.x, m.x, tab.one_minus_mu), m.y = muon_momentum(g.y, m.y, tab.one_minus_mu);
        m.z = muon_momentum(g.z, m.z, tab.one_minus_mu), m.w = muon_momentum(g.w, m.w, tab.one_minus_mu);
        return make_float4(muon_update(g.x, m.x, tab.mu, tab.nesterov), muon_update(g.y, m.y, tab.mu, tab.nesterov),
                           muon_update(g.z, m.z, tab.mu, tab.nesterov), muon_update(g.w, m.w, tab.mu, tab.nesterov));
    };
    constexpr int U = 4; // moves on their way at once

    if (tid == 0) {
        mbar_init(&done, 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)),
                     "r"(sh.columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // zeros: rows past m, columns past the slab
    for (int i = tid; i < (2 * x_plane + 2 * a_plane) / 16; i += kClusterThreads)
        reinterpret_cast<uint4 *>(base)[i] = make_uint4(0, 0, 0, 0);
    // the norm: sums in 64 bits, in a fixed order
    double s = 0.0;
    float4 g0[U], m0[U]; // the first turn's values stay for the second pass, which is all of a small slab
    for (int e0 = tid; e0 < moves; e0 += U * kClusterThreads) {
        float4 g[U], m[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * kClusterThreads;
            int i, j;
            g[u] = m[u] = make_float4(0, 0, 0, 0);
            if (e < moves) g[u] = fetch(place(e, i, j), e < fours, m[u]);
            if (e0 == tid) g0[u] = g[u], m0[u] = m[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4 w = updated(g[u], m[u]);
            s = fma((double)w.x, (double)w.x, s);
            s = fma((double)w.y, (double)w.y, s);
            s = fma((double)w.z, (double)w.z, s);
            s = fma((double)w.w, (double)w.w, s);
        }
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) warp_sum[warp] = s;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_at, 0);
    s = 0.0;
    for (int w = 0; w < kClusterThreads / 32; ++w) s += warp_sum[w];
    if (sh.blocks > 1) {
        if (tid == 0) block_total = s;
        cluster_sync();
        s = 0.0;
        for (int r = 0; r < sh.blocks; ++r) s += remote_load_f64(remote(smem_u32(&block_total), r));
    }
    const double norm = sqrt(s);
    const Divisor d = divisor_of(norm, eps);
    auto put = [&](int i, int j, float v) {
        v = v * d.pre / d.div * sh.x_scale;
        const __half h = __float2half_rn(v);
        const uint32_t p = plane_byte(sh.m16, i, j);
        *reinterpret_cast<__half *>(x_hi + p) = h;
        *reinterpret_cast<__half *>(x_lo + p) = __float2half_rn(v - __half2float(h));
    };
    for (int e0 = tid; e0 < moves; e0 += U * kClusterThreads) {
        float4 g[U], m[U];
        size_t at[U];
        int i[U], j[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * kClusterThreads;
            if (e < moves) {
                at[u] = place(e, i[u], j[u]);
                if (e0 == tid) g[u] = g0[u], m[u] = m0[u];
                else g[u] = fetch(at[u], e < fours, m[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * kClusterThreads;
            if (e >= moves) continue;
            const float4 w = updated(g[u], m[u]);
            put(i[u], j[u], w.x);
            if (e < fours) {
                if (MUON) *reinterpret_cast<VM *>(mom + at[u]) = Quad<M>::put(m[u]);
                next(i[u], j[u]);
                put(i[u], j[u], w.y);
                next(i[u], j[u]);
                put(i[u], j[u], w.z);
                next(i[u], j[u]);
                put(i[u], j[u], w.w);
            } else if (MUON) {
                mom[at[u]] = from_f32<M>(m[u].x);
            }
        }
    }

    const bool keep = !MUON && kept.x.hi != nullptr;
    if (keep && tid == 0 && rank == 0) kept.norms[b] = d.small ? -1.0 : norm;
    // rows [r0, r1) and columns up to `used` of a plane pair to memory, 16 bytes at a time
    auto dump = [&](const char *hi, const char *lo, const OrthoPlanes &to, int step, int r0, int r1, int used, int col0) {
        const int eights = (used + 7) / 8;
        __half *out = to.hi + step * kept.step + (size_t)b * to.stride;
        const ptrdiff_t to_lo = to.lo - to.hi;
        for (int t = tid; t < (r1 - r0) * eights; t += kClusterThreads) {
            const int i = r0 + t / eights, c = (t - (i - r0) * eights) * 8;
            const uint32_t from = plane_byte(sh.m16, i, c);
            uint4 *at = reinterpret_cast<uint4 *>(out + (size_t)i * to.ld + col0 + c);
            *at = *reinterpret_cast<const uint4 *>(hi + from);
            *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(at) + to_lo) = *reinterpret_cast<const uint4 *>(lo + from);
        }
    };
    const int own0 = sh.blocks > 1 ? min(sh.m, (int)rank * sh.per) : 0, own1 = sh.blocks > 1 ? min(sh.m, own0 + sh.per) : sh.m;

    const int row = 32 * (warp % 4) + lane, turn = warp / 4; // columns 16 (turn + 4 k) ..
    const uint32_t acc = tmem + ((uint32_t)(32 * (warp % 4)) << 16);
    const bool rows_here = 32 * (warp % 4) < sh.m16; // the warp has rows (all its lanes read TMEM together)
    const bool mine = row < sh.m16;
    const uint32_t xh = smem_u32(x_hi), xl = smem_u32(x_lo), ah = smem_u32(a_hi), al = smem_u32(a_lo);
    const int ns16 = (sh.ns + 15) / 16 * 16;
    const uint32_t leader = elect_leader();
    const Operands gram = operands(xh, xl, xh, xl, sh.m16, true), square = operands(ah, al, ah, al, sh.m16, true),
                   apply = operands(ah, al, xh, xl, sh.m16, false);
    const uint32_t idesc_a = mma_desc(sh.m16, true);
    uint32_t phase = 0;
    // what was written to shared memory is multiplied, and every thread waits for the product
    auto begin = [&] {
        async_proxy_fence();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    auto finish = [&] {
        if (!*abort) mbar_wait(&done, phase, abort);
        phase ^= 1u;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    for (int step = 0; step < co.n; ++step) {
        const float *cf = co.c[step];
        // A
        begin();
        if (warp == 0) {
            multiply(tmem, gram, idesc_a, ns16, leader);
            mma_commit(&done, leader);
        }
        if (keep) dump(x_hi, x_lo, kept.x, step, 0, sh.m, cols, j0);
        const uint32_t owner = mine ? row / sh.per : 0; // of this row of A
        const uint32_t to = sh.blocks > 1 ? remote(smem_u32(partial) + ((int)rank * (sh.m16 / 4) * sh.per + row - (int)owner * sh.per) * 16, owner) : 0u;
        finish();
        if (rows_here)
            for (int c = 16 * turn; c < sh.m16; c += 64) {
                float v[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
                if (sh.blocks > 1) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        remote_store4(to + (c / 4 + k) * sh.per * 16, make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]),
                                                                       __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3])));
                } else {
                    float on = 0.f;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        on = c + k == row ? v[k] : on;
                        v[k] = c + k == row ? 0.f : v[k] * sh.to_a;
                    }
                    if ((row & ~15) == c) diag_a[row] = on * sh.to_d;
                    planes_put16(a_hi, a_lo, sh.m16, row, c, v);
                }
            }
        if (sh.blocks > 1) {
            if (*abort) { // a wait of this block ran out: the others' A will be wrong too
                for (int r = 0; r < sh.blocks; ++r) remote_store_f32(remote(smem_u32(&abort_flag), r), __int_as_float(1));
            }
            cluster_sync();
            // add up this block's rows, in the order of the blocks, then give them to all
            const int r0 = (int)rank * sh.per, rows = max(0, min(sh.m16, r0 + sh.per) - r0), pieces = rows * (sh.m16 / 8);
            for (int t = tid; t < pieces; t += kClusterThreads) {
                const int c8 = t / rows, i = t - c8 * rows, c = c8 * 8;
                float v[8] = {};
#pragma unroll 8
                for (int r = 0; r < sh.blocks; ++r) {
                    const float4 *p = reinterpret_cast<const float4 *>(partial) + (r * (sh.m16 / 4) + c / 4) * sh.per + i;
                    const float4 f = p[0], g = p[sh.per];
                    v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
                    v[4] += g.x, v[5] += g.y, v[6] += g.z, v[7] += g.w;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (c + k == r0 + i) diag_a[r0 + i] = v[k] * sh.to_d;
                    v[k] = c + k == r0 + i ? 0.f : v[k] * sh.to_a;
                }
                uint4 hi, lo;
                split8(v, hi, lo);
                const uint32_t at = plane_byte(sh.m16, r0 + i, c);
                *reinterpret_cast<uint4 *>(a_hi + at) = hi;
                *reinterpret_cast<uint4 *>(a_lo + at) = lo;
            }
            __syncthreads();
            // as they lie: 128 bytes of a row, then the next row's, so that a warp's pieces reach the other block together
            const int line = rows * 128, all = 2 * (sh.mk / 64) * line; // bytes of a plane's block of 64 columns; of both planes'
            for (int u = tid * 16; u < all; u += kClusterThreads * 16) {
                int rest = u, offset = r0 * 128;
                while (rest >= line) rest -= line, offset += sh.m16 * 128; // at most 3 times: lo follows hi
                const uint32_t at = offset + rest;
                const uint4 piece = *reinterpret_cast<const uint4 *>(a_hi + at);
#pragma unroll
                for (int o = 1; o < kClusterMax; ++o)
                    if (o < sh.blocks) remote_store4(remote(ah + at, (rank + o) & (sh.blocks - 1)), piece);
            }
            if (tid < rows)
                for (int o = 1; o < sh.blocks; ++o)
                    remote_store_f32(remote(smem_u32(&diag_a[r0 + tid]), (rank + o) & (sh.blocks - 1)), diag_a[r0 + tid]);
            asm volatile("fence.proxy.async.shared::cluster;" ::: "memory");
            cluster_sync();
        }
        // B
        begin();
        if (warp == 0) {
            multiply(tmem, square, idesc_a, sh.m16, leader);
            mma_commit(&done, leader);
        }
        if (keep) {
            dump(a_hi, a_lo, kept.a, step, own0, own1, sh.m, 0);
            if (rank == 0 && tid < sh.m)
                reinterpret_cast<float *>(reinterpret_cast<__half *>(kept.da) + step * kept.step)[(size_t)b * sh.m + tid] = diag_a[tid];
            __syncthreads(); // B takes A's place
        }
        float o[16];
        float di = 0.f;
        if (mine) {
            di = diag_a[row];
            if (16 * turn < sh.m16) planes_get16(a_hi, a_lo, sh.m16, row, 16 * turn, o);
        }
        finish();
        if (rows_here)
            for (int c = 16 * turn; c < sh.m16; c += 64) {
                float v[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
                const float base = fmaf(cf[2], di, cf[1]);
                float on = 0.f; // the diagonal's sum
#pragma unroll
                for (int k4 = 0; k4 < 16; k4 += 4) {
                    const float4 dj = *reinterpret_cast<const float4 *>(diag_a + c + k4);
                    const float d4[4] = {dj.x, dj.y, dj.z, dj.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = k4 + i;
                        const float w = fmaf(fmaf(cf[2], d4[i], base), o[k], cf[3] * v[k]);
                        on = c + k == row ? v[k] : on;
                        v[k] = c + k == row ? 0.f : w;
                    }
                }
                if ((row & ~15) == c) diag_b[row] = fmaf(cf[4], di, fmaf(cf[5] * di, di, cf[6] * on));
                planes_put16(a_hi, a_lo, sh.m16, row, c, v);
                if (c + 64 < sh.m16) planes_get16(a_hi, a_lo, sh.m16, row, c + 64, o);
            }
        // X
        begin();
        if (warp == 0) {
            Operands part = apply;
            for (int c = 0; c < ns16; c += 256) {
                multiply(tmem + c, part, mma_desc(min(256, ns16 - c), false), sh.m16, leader);
                part.q += 4 * part.p_block, part.q_lo += 4 * part.p_block; // four blocks of 64 columns on
            }
            mma_commit(&done, leader);
        }
        if (keep) {
            dump(a_hi, a_lo, kept.b, step, own0, own1, sh.m, 0);
            if (rank == 0 && tid < sh.m)
                reinterpret_cast<float *>(reinterpret_cast<__half *>(kept.db) + step * kept.step)[(size_t)b * sh.m + tid] = diag_b[tid];
        }
        float f = 0.f;
        if (mine) {
            f = cf[0] + diag_b[row];
            if (16 * turn < ns16) planes_get16(x_hi, x_lo, sh.m16, row, 16 * turn, o);
        }
        finish();
        if (rows_here) {
            const bool last = step + 1 == co.n;
            for (int c = 16 * turn; c < ns16; c += 64) {
                float v[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = fmaf(f, o[k], sh.unscale_b * v[k]);
                if (c + 64 < ns16) planes_get16(x_hi, x_lo, sh.m16, row, c + 64, o);
                if (!last) {
                    planes_put16(x_hi, x_lo, sh.m16, row, c, v);
                } else { // the result itself, 32-bit, in the place of the two planes: hi 0..3, 4..7, lo 8..11, 12..15
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t at = plane_byte(sh.m16, row, c + 8 * h);
                        const float u = sh.unscale_x;
                        *reinterpret_cast<float4 *>(x_hi + at) = make_float4(v[4 * h] * u, v[4 * h + 1] * u, v[4 * h + 2] * u, v[4 * h + 3] * u);
                        *reinterpret_cast<float4 *>(x_lo + at) = make_float4(v[8 + 4 * h] * u, v[9 + 4 * h] * u, v[10 + 4 * h] * u, v[11 + 4 * h] * u);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const bool poisoned = *abort != 0; // a wait ran out
    for (int i = 0; poisoned && i < 10000; ++i) __nanosleep(1000); // the products in flight end within this time
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(sh.columns) : "memory");
    if (keep && poisoned && tid == 0) kept.norms[b] = NAN; // for the backward pass
    auto get = [&](int i, int j) -> float {
        const int w = j & 15;
        const float v = *reinterpret_cast<const float *>((w < 8 ? x_hi : x_lo) + plane_byte(sh.m16, i, (j & ~15) + ((w >> 2) & 1) * 8) + (w & 3) * 4);
        return poisoned ? NAN : v;
    };
    for (int e0 = tid; e0 < moves; e0 += U * kClusterThreads) {
        float4 p[U];
        size_t at[U];
        int i[U], j[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * kClusterThreads;
            if (e < moves) {
                at[u] = place(e, i[u], j[u]);
                if (MUON) {
                    const T *q = static_cast<const T *>(tab.param[tensor]) + mat + at[u];
                    if (e < fours) p[u] = Quad<T>::get(*reinterpret_cast<const VT *>(q));
                    else p[u].x = to_f32(*q);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int e = e0 + u * kClusterThreads;
            if (e >= moves) continue;
            float4 v = {};
            v.x = get(i[u], j[u]);
            if (e < fours) {
                next(i[u], j[u]);
                v.y = get(i[u], j[u]);
                next(i[u], j[u]);
                v.z = get(i[u], j[u]);
                next(i[u], j[u]);
                v.w = get(i[u], j[u]);
            }
            T *out = (MUON ? static_cast<T *>(tab.param[tensor]) : y) + mat + at[u];
            if (MUON) {
                const float lr = tab.lr[tensor], decay = tab.decay[tensor];
                v = make_float4(muon_param(p[u].x, v.x, lr, decay), muon_param(p[u].y, v.y, lr, decay),
                                muon_param(p[u].z, v.z, lr, decay), muon_param(p[u].w, v.w, lr, decay));
            }
            if (e < fours) *reinterpret_cast<VT *>(out) = Quad<T>::put(v);
            else *out = from_f32<T>(v.x);
        }
    }
}

static ClusterShape cluster_shape(int rows, int cols, int blocks) {
    ClusterShape s = {};
    s.m = std::min(rows, cols);
    s.n = std::max(rows, cols);
    s.transposed = rows > cols;
    s.m16 = (s.m + 15) / 16 * 16;
    s.mk = (s.m16 + 63) / 64 * 64;
    s.blocks = blocks;
    s.ns = ((s.n + blocks - 1) / blocks + 15) / 16 * 16;
    s.ns64 = (s.ns + 63) / 64 * 64;
    s.per = (s.m16 + blocks - 1) / blocks;
    s.columns = 32;
    while (s.columns < std::max(s.m16, s.ns)) s.columns *= 2;
    const size_t planes = 4 * (size_t)s.m16 * (s.ns64 + s.mk);
    // a 128-row operand reads past a plane of fewer rows: into what follows, whose rows of the product are not read
    size_t smem = 1024 + planes + std::max<size_t>(blocks > 1 ? 4 * (size_t)s.per * blocks * s.m16 : 0, (size_t)(128 - s.m16) * 128);
    // blocks that share an SM must find their TMEM columns free: as large a part of its shared memory as of its TMEM
    smem = std::max(smem, kClusterSmem * s.columns / 512 - kClusterStatic);
    s.smem = smem;
    return s;
}

static bool cluster_fits(const ClusterShape &s) { return s.columns <= 512 && s.smem + kClusterStatic <= kClusterSmem; }

// The blocks of a cluster for a matrix, or 0 where it does not fit.
static int cluster_blocks(int rows, int cols) {
    if (std::min(rows, cols) > kClusterMaxShort || std::max(rows, cols) > 512 * kClusterMax) return 0; // 512 columns of TMEM a block
    for (int c = 1; c <= kClusterMax; c *= 2)
        if (cluster_fits(cluster_shape(rows, cols, c))) return c;
    return 0;
}

int ortho_is_clustered(int rows, int cols) { return cluster_blocks(rows, cols); }

template <typename T, typename M, bool MUON>
static int cluster_launch(long long batch, const ClusterShapes<MUON> &shapes, size_t smem, const void *x, void *y, const MuonTable &tab,
                          const ClusterSteps &steps, float eps, const ClusterKept &kept, cudaStream_t stream) {
    auto *kernel = ortho_cluster_kernel<T, M, MUON>;
    const int blocks = shapes.of[0].blocks;
    if (batch * blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "orthogonalize: too many matrices");
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch("ortho_cluster_kernel attributes");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * blocks));
    cfg.blockDim = dim3(kClusterThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, shapes, static_cast<const T *>(x), static_cast<T *>(y), tab, steps, eps, kept);
    if (e != cudaSuccess) return set_error(kErrLaunch, "ortho_cluster_kernel: %s", cudaGetErrorString(e));
    return check_launch("ortho_cluster_kernel");
}

// More blocks a cluster than a matrix needs, where there are SMs for them and a block's slab stays at least 128
// columns: below that the exchange of A costs more than the shorter slab saves ([128, 128] 54 us in one
// block, 72 in two; [64, 512] 77 us in one, 56 in four).
static int cluster_widen(const int sizes[][2], int n, long long batch) {
    int blocks = cluster_blocks(sizes[0][0], sizes[0][1]), sms = 148, dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    auto wide = [&] {
        for (int i = 0; i < n; ++i)
            if (cluster_shape(sizes[i][0], sizes[i][1], blocks).ns < 256) return false;
        return true;
    };
    while (2 * blocks <= kClusterMax && batch * 2 * blocks <= sms && wide()) blocks *= 2;
    return blocks;
}

static ClusterShape cluster_plan(int rows, int cols, int blocks, float x_scale, float a_scale, float b_scale) {
    ClusterShape sh = cluster_shape(rows, cols, blocks);
    sh.x_scale = x_scale;
    sh.to_a = a_scale / (x_scale * x_scale);
    sh.to_d = 1.f / (x_scale * x_scale);
    sh.unscale_b = 1.f / b_scale;
    sh.unscale_x = 1.f / x_scale;
    return sh;
}
static ClusterSteps cluster_steps(const OrthoCoefficients &co, float a_scale, float b_scale) {
    ClusterSteps steps = {};
    steps.n = co.steps;
    for (int k = 0; k < co.steps; ++k) {
        const float a = co.c[k][0], b = co.c[k][1], c = co.c[k][2];
        const float v[7] = {a, b * (b_scale / a_scale), c * (b_scale / a_scale), c * (b_scale / (a_scale * a_scale)), b, c,
                            c / (a_scale * a_scale)};
        std::copy(v, v + 7, steps.c[k]);
    }
    return steps;
}

int ortho_cluster_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y, const OrthoCoefficients &co,
                      float x_scale, float a_scale, float b_scale, float eps, const ClusterKept &kept, cudaStream_t stream) {
    ClusterShapes<false> sh = {};
    const int sizes[1][2] = {{rows, cols}};
    sh.of[0] = cluster_plan(rows, cols, cluster_widen(sizes, 1, batch), x_scale, a_scale, b_scale);
    const ClusterSteps st = cluster_steps(co, a_scale, b_scale);
    static const MuonTable none = {};
    const size_t smem = sh.of[0].smem;
    if (dtype == kOrthoF32) return cluster_launch<float, float, false>(batch, sh, smem, x, y, none, st, eps, kept, stream);
    if (dtype == kOrthoBF16) return cluster_launch<__nv_bfloat16, float, false>(batch, sh, smem, x, y, none, st, eps, kept, stream);
    return cluster_launch<__half, float, false>(batch, sh, smem, x, y, none, st, eps, kept, stream);
}

int ortho_cluster_muon(const MuonTable &t, const int sizes[][2], const OrthoCoefficients &co, float x_scale, float a_scale, float b_scale,
                       float eps, cudaStream_t stream) {
    ClusterShapes<true> sh = {};
    size_t smem = 0;
    const int blocks = cluster_widen(sizes, t.n, t.first[t.n]);
    for (int i = 0; i < t.n; ++i) {
        sh.of[i] = cluster_plan(sizes[i][0], sizes[i][1], blocks, x_scale, a_scale, b_scale);
        smem = std::max(smem, sh.of[i].smem);
    }
    const ClusterSteps st = cluster_steps(co, a_scale, b_scale);
    const ClusterKept none = {};
    const long long batch = t.first[t.n];
    const bool same = t.dtype == t.state_dtype;
    if (t.dtype == kOrthoF32) return cluster_launch<float, float, true>(batch, sh, smem, nullptr, nullptr, t, st, eps, none, stream);
    if (t.dtype == kOrthoBF16)
        return same ? cluster_launch<__nv_bfloat16, __nv_bfloat16, true>(batch, sh, smem, nullptr, nullptr, t, st, eps, none, stream)
                    : cluster_launch<__nv_bfloat16, float, true>(batch, sh, smem, nullptr, nullptr, t, st, eps, none, stream);
    return same ? cluster_launch<__half, __half, true>(batch, sh, smem, nullptr, nullptr, t, st, eps, none, stream)
                : cluster_launch<__half, float, true>(batch, sh, smem, nullptr, nullptr, t, st, eps, none, stream);
}

} // namespace gsb
