// Newton-Schulz steps of matrices whose short side is at most 128, in one launch: a
// cluster of blocks holds a matrix X [m, n] in shared memory, each block a slab of its columns, from
// the first read to the last write.
//
// What bounds such a matrix is not its products but the chain of them: 15 launches of
// the tiled kernel took 165 us for a stack of 64 x 64. Here a step is
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
    int slack;              // bytes behind the planes that a 128-row operand may touch
    float x_scale, a_scale, b_scale;
    size_t smem;
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
__device__ __forceinline__ float4 remote_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
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
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }

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

// One thread: D[128, n] = P Q over `depth`, hi and lo planes of both; P and Q depth-major from their
// first row (X X^T, A A), or Q column-major (B X). `rows`: of the planes.
__device__ __forceinline__ void multiply(uint32_t d, uint32_t p, uint32_t p_lo, uint32_t q, uint32_t q_lo, int rows_p,
                                         int rows_q, bool q_k_major, int n, int depth) {
    const uint32_t idesc = mma_desc(n, q_k_major);
    const uint32_t chunk_p = rows_p * 128, chunk_q = rows_q * 128;
    for (int k = 0; k < depth; k += 16) {
        const uint32_t po = (k >> 6) * chunk_p + ((k >> 4) & 3) * 32;
        const uint32_t qo = q_k_major ? (k >> 6) * chunk_q + ((k >> 4) & 3) * 32 : k * 128;
        const uint64_t ph = operand_desc(p + po, true, 0), pl = operand_desc(p_lo + po, true, 0);
        const uint64_t qh = operand_desc(q + qo, q_k_major, chunk_q), ql = operand_desc(q_lo + qo, q_k_major, chunk_q);
        mma_f16(d, ph, qh, idesc, k > 0);
        mma_f16(d, ph, ql, idesc, true);
        mma_f16(d, pl, qh, idesc, true);
    }
}

template <typename T, typename M, bool MUON>
__global__ void __launch_bounds__(kClusterThreads, 1)
    ortho_cluster_kernel(const __grid_constant__ ClusterShape sh, const T *x_in, T *y, const __grid_constant__ MuonTable tab,
                         const __grid_constant__ OrthoCoefficients co, float eps) {
    extern __shared__ char raw[];
    __shared__ float diag_a[kClusterMaxShort], diag_b[kClusterMaxShort];
    __shared__ double warp_sum[kClusterThreads / 32], block_total;
    __shared__ alignas(8) unsigned long long done;
    __shared__ uint32_t tmem_at;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t rank = sh.blocks > 1 ? cluster_rank() : 0;
    const long long b = blockIdx.x / sh.blocks;
    const int tensor = MUON ? muon_tensor_of(tab, b) : 0;
    if (MUON && !muon_visible(tab, tensor, b)) return; // the whole cluster alike

    char *base = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int x_plane = sh.m16 * sh.ns64 * 2, a_plane = sh.m16 * sh.mk * 2;
    char *x_hi = base, *x_lo = x_hi + x_plane, *a_hi = x_lo + x_plane, *a_lo = a_hi + a_plane;
    float *partial = reinterpret_cast<float *>(a_lo + a_plane); // several blocks: [m16, m16 + 4]
    const int pitch = sh.m16 + 4;
    volatile int *abort = &abort_flag;

    const int j0 = (int)rank * sh.ns, cols = max(0, min(sh.ns, sh.n - j0)); // this block's columns
    const size_t numel = (size_t)sh.m * sh.n;
    const size_t mat = (size_t)(MUON ? b - tab.first[tensor] : b) * numel;
    const T *grad = MUON ? static_cast<const T *>(tab.grad[tensor]) + mat : x_in + mat;
    M *mom = MUON ? static_cast<M *>(tab.momentum[tensor]) + mat : nullptr;
    // value e of the block's slab, in the tensor's order: its place there, its row and column here
    const int inner = sh.transposed ? sh.m : cols, count = sh.m * cols;
    auto place = [&](int e, int &i, int &j) -> size_t {
        const int o = e / inner, k = e - o * inner;
        i = sh.transposed ? k : o;
        j = sh.transposed ? o : k;
        return sh.transposed ? (size_t)(j0 + o) * sh.m + k : (size_t)o * sh.n + j0 + k;
    };

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
#pragma unroll 4
    for (int e = tid; e < count; e += kClusterThreads) {
        int i, j;
        const size_t at = place(e, i, j);
        float v = to_f32(grad[at]);
        if (MUON) v = muon_update(v, muon_momentum(v, to_f32(mom[at]), tab.one_minus_mu), tab.mu, tab.nesterov);
        s = fma((double)v, (double)v, s);
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) warp_sum[warp] = s;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_at;
    s = 0.0;
    for (int w = 0; w < kClusterThreads / 32; ++w) s += warp_sum[w];
    if (sh.blocks > 1) {
        if (tid == 0) block_total = s;
        cluster_sync();
        s = 0.0;
        for (int r = 0; r < sh.blocks; ++r) s += remote_load_f64(remote(smem_u32(&block_total), r));
    }
    const float norm = (float)sqrt(s), div = norm < eps ? eps : norm;
#pragma unroll 4
    for (int e = tid; e < count; e += kClusterThreads) {
        int i, j;
        const size_t at = place(e, i, j);
        float v = to_f32(grad[at]);
        if (MUON) {
            const float m = muon_momentum(v, to_f32(mom[at]), tab.one_minus_mu);
            mom[at] = from_f32<M>(m);
            v = muon_update(v, m, tab.mu, tab.nesterov);
        }
        v = v / div * sh.x_scale;
        const __half h = __float2half_rn(v);
        const uint32_t p = plane_byte(sh.m16, i, j);
        *reinterpret_cast<__half *>(x_hi + p) = h;
        *reinterpret_cast<__half *>(x_lo + p) = __float2half_rn(v - __half2float(h));
    }

    const int row = 32 * (warp % 4) + lane, turn = warp / 4; // columns 16 (turn + 4 k) ..
    const uint32_t acc = tmem + ((uint32_t)(32 * (warp % 4)) << 16);
    const bool rows_here = 32 * (warp % 4) < sh.m16; // the warp has rows (all its lanes read TMEM together)
    const bool mine = row < sh.m16;
    const uint32_t xh = smem_u32(x_hi), xl = smem_u32(x_lo), ah = smem_u32(a_hi), al = smem_u32(a_lo);
    const int ns16 = (sh.ns + 15) / 16 * 16;
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
    for (int step = 0; step < co.steps; ++step) {
        const float ca = co.c[step][0], cb = co.c[step][1], cc = co.c[step][2];
        // A
        begin();
        if (tid == 0) {
            multiply(tmem, xh, xl, xh, xl, sh.m16, sh.m16, true, sh.m16, ns16);
            mma_commit(&done);
        }
        finish();
        const float to_a = sh.a_scale / (sh.x_scale * sh.x_scale), to_d = 1.f / (sh.x_scale * sh.x_scale);
        if (rows_here)
            for (int c = 16 * turn; c < sh.m16; c += 64) {
                float v[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
                if (sh.blocks > 1) {
                    float4 *p = reinterpret_cast<float4 *>(partial + row * pitch + c);
#pragma unroll
                    for (int k = 0; k < 4; ++k) p[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        if (c + k == row) diag_a[row] = v[k] * to_d;
                        v[k] = c + k == row ? 0.f : v[k] * to_a;
                    }
                    planes_put16(a_hi, a_lo, sh.m16, row, c, v);
                }
            }
        if (sh.blocks > 1) {
            cluster_sync();
            const int per = (sh.m16 + sh.blocks - 1) / sh.blocks, r0 = (int)rank * per, r1 = min(sh.m16, r0 + per);
            const int eights = sh.m16 / 8;
            for (int t = tid; t < (r1 - r0) * eights; t += kClusterThreads) {
                const int i = r0 + t / eights, c = (t % eights) * 8;
                float v[8] = {};
                for (int r = 0; r < sh.blocks; ++r) {
                    const uint32_t p = remote(smem_u32(partial + i * pitch + c), r);
                    const float4 f = remote_load4(p), g = remote_load4(p + 16);
                    v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
                    v[4] += g.x, v[5] += g.y, v[6] += g.z, v[7] += g.w;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (c + k == i)
                        for (int r = 0; r < sh.blocks; ++r) remote_store_f32(remote(smem_u32(&diag_a[i]), r), v[k] * to_d);
                    v[k] = c + k == i ? 0.f : v[k] * to_a;
                }
                uint4 hi, lo;
                split8(v, hi, lo);
                const uint32_t at = plane_byte(sh.m16, i, c);
                for (int r = 0; r < sh.blocks; ++r) {
                    remote_store4(remote(ah + at, r), hi);
                    remote_store4(remote(al + at, r), lo);
                }
            }
            async_proxy_fence();
            cluster_sync();
        }
        // B
        begin();
        if (tid == 0) {
            multiply(tmem, ah, al, ah, al, sh.m16, sh.m16, true, sh.m16, sh.m16);
            mma_commit(&done);
        }
        finish();
        if (rows_here) {
            const float di = mine ? diag_a[row] : 0.f;
            const float c0 = cb * (sh.b_scale / sh.a_scale), c1 = cc * (sh.b_scale / sh.a_scale),
                        c2 = cc * (sh.b_scale / (sh.a_scale * sh.a_scale)), c5 = cc / (sh.a_scale * sh.a_scale);
            for (int c = 16 * turn; c < sh.m16; c += 64) {
                float v[16], o[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
                planes_get16(a_hi, a_lo, sh.m16, row, c, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (c + k == row) {
                        diag_b[row] = fmaf(cb, di, fmaf(cc * di, di, c5 * v[k]));
                        v[k] = 0.f;
                    } else {
                        v[k] = fmaf(fmaf(c1, di + diag_a[c + k], c0), o[k], c2 * v[k]);
                    }
                }
                planes_put16(a_hi, a_lo, sh.m16, row, c, v);
            }
        }
        // X
        begin();
        if (tid == 0) {
            for (int c = 0; c < ns16; c += 256)
                multiply(tmem + c, ah, al, xh + (c >> 6) * sh.m16 * 128, xl + (c >> 6) * sh.m16 * 128, sh.m16, sh.m16, false,
                         min(256, ns16 - c), sh.m16);
            mma_commit(&done);
        }
        finish();
        if (rows_here) {
            const bool last = step + 1 == co.steps;
            const float f = ca + (mine ? diag_b[row] : 0.f), unscale = 1.f / sh.b_scale, out = 1.f / sh.x_scale;
            for (int c = 16 * turn; c < ns16; c += 64) {
                float v[16], o[16];
                __syncwarp();
                tmem_load16(acc + c, v);
                if (!mine) continue;
                planes_get16(x_hi, x_lo, sh.m16, row, c, o);
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = fmaf(f, o[k], unscale * v[k]);
                if (!last) {
                    planes_put16(x_hi, x_lo, sh.m16, row, c, v);
                } else { // the result itself, 32-bit, in the place of the two planes: hi 0..3, 4..7, lo 8..11, 12..15
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t at = plane_byte(sh.m16, row, c + 8 * h);
                        *reinterpret_cast<float4 *>(x_hi + at) =
                            make_float4(v[4 * h] * out, v[4 * h + 1] * out, v[4 * h + 2] * out, v[4 * h + 3] * out);
                        *reinterpret_cast<float4 *>(x_lo + at) =
                            make_float4(v[8 + 4 * h] * out, v[9 + 4 * h] * out, v[10 + 4 * h] * out, v[11 + 4 * h] * out);
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(sh.columns) : "memory");
    const bool poisoned = *abort != 0; // a wait ran out
#pragma unroll 4
    for (int e = tid; e < count; e += kClusterThreads) {
        int i, j;
        const size_t at = place(e, i, j);
        const int w = j & 15;
        const char *plane = w < 8 ? x_hi : x_lo;
        float v = *reinterpret_cast<const float *>(plane + plane_byte(sh.m16, i, (j & ~15) + ((w >> 2) & 1) * 8) + (w & 3) * 4);
        if (poisoned) v = NAN;
        if (MUON) {
            T *p = static_cast<T *>(tab.param[tensor]) + mat + at;
            *p = from_f32<T>(muon_param(to_f32(*p), v, tab.lr[tensor], tab.decay[tensor]));
        } else {
            y[mat + at] = from_f32<T>(v);
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
    s.columns = 32;
    while (s.columns < std::max(s.m16, s.ns)) s.columns *= 2;
    const size_t planes = 4 * (size_t)s.m16 * (s.ns64 + s.mk);
    // a 128-row operand reads past a plane of fewer rows: into what follows, whose rows of the product are not read
    size_t smem = 1024 + planes + std::max<size_t>(blocks > 1 ? 4 * (size_t)s.m16 * (s.m16 + 4) : 0, (size_t)(128 - s.m16) * 128);
    // blocks that share an SM must find their TMEM columns free: as large a part of its shared memory as of its TMEM
    smem = std::max(smem, kClusterSmem * s.columns / 512 - kClusterStatic);
    s.smem = smem;
    return s;
}

static bool cluster_fits(const ClusterShape &s) { return s.columns <= 512 && s.smem + kClusterStatic <= kClusterSmem; }

// The blocks of a cluster for a matrix, or 0 where it does not fit.
static int cluster_blocks(int rows, int cols) {
    if (std::min(rows, cols) > kClusterMaxShort) return 0;
    for (int c = 1; c <= kClusterMax; c *= 2)
        if (cluster_fits(cluster_shape(rows, cols, c))) return c;
    return 0;
}

bool ortho_is_clustered(int rows, int cols) { return cluster_blocks(rows, cols) > 0; }

template <typename T, typename M, bool MUON>
static int cluster_launch(long long batch, const ClusterShape &sh, const void *x, void *y, const MuonTable &tab,
                          const OrthoCoefficients &co, float eps, cudaStream_t stream) {
    auto *kernel = ortho_cluster_kernel<T, M, MUON>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sh.smem) != cudaSuccess)
        return check_launch("ortho_cluster_kernel attributes");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * sh.blocks));
    cfg.blockDim = dim3(kClusterThreads);
    cfg.dynamicSmemBytes = sh.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = sh.blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, sh, static_cast<const T *>(x), static_cast<T *>(y), tab, co, eps);
    if (e != cudaSuccess) return set_error(kErrLaunch, "ortho_cluster_kernel: %s", cudaGetErrorString(e));
    return check_launch("ortho_cluster_kernel");
}

static int cluster_shape_for(const char *what, long long batch, int rows, int cols, float x_scale, float a_scale, float b_scale, ClusterShape *sh) {
    *sh = cluster_shape(rows, cols, cluster_blocks(rows, cols));
    sh->x_scale = x_scale;
    sh->a_scale = a_scale;
    sh->b_scale = b_scale;
    if (batch * sh->blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "%s: too many matrices", what);
    return kOk;
}

int ortho_cluster_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y, const OrthoCoefficients &co,
                      float x_scale, float a_scale, float b_scale, float eps, cudaStream_t stream) {
    ClusterShape sh;
    if (int e = cluster_shape_for("orthogonalize", batch, rows, cols, x_scale, a_scale, b_scale, &sh)) return e;
    static const MuonTable none = {};
    if (dtype == kOrthoF32) return cluster_launch<float, float, false>(batch, sh, x, y, none, co, eps, stream);
    if (dtype == kOrthoBF16) return cluster_launch<__nv_bfloat16, float, false>(batch, sh, x, y, none, co, eps, stream);
    return cluster_launch<__half, float, false>(batch, sh, x, y, none, co, eps, stream);
}

int ortho_cluster_muon(const MuonTable &t, int rows, int cols, const OrthoCoefficients &co, float x_scale, float a_scale,
                       float b_scale, float eps, cudaStream_t stream) {
    ClusterShape sh;
    const long long batch = t.first[t.n];
    if (int e = cluster_shape_for("muon", batch, rows, cols, x_scale, a_scale, b_scale, &sh)) return e;
    const bool same = t.dtype == t.state_dtype;
    if (t.dtype == kOrthoF32) return cluster_launch<float, float, true>(batch, sh, nullptr, nullptr, t, co, eps, stream);
    if (t.dtype == kOrthoBF16)
        return same ? cluster_launch<__nv_bfloat16, __nv_bfloat16, true>(batch, sh, nullptr, nullptr, t, co, eps, stream)
                    : cluster_launch<__nv_bfloat16, float, true>(batch, sh, nullptr, nullptr, t, co, eps, stream);
    return same ? cluster_launch<__half, __half, true>(batch, sh, nullptr, nullptr, t, co, eps, stream)
                : cluster_launch<__half, float, true>(batch, sh, nullptr, nullptr, t, co, eps, stream);
}

} // namespace gsb
