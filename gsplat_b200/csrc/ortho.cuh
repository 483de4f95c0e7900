// Shared declarations of the matrix-orthogonalising operators (orthogonalize.cu,
// ortho_thin.cu, ortho_gemm.cu).
//
// X0 = U / max(|U|_F, eps), then for every step (a, b, c)
//     A = X X^T,  B = b A + c A A,  X <- a X + B X
// on the orientation whose rows are the shorter side (a tall U is transposed:
// the iteration commutes with transposition).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "gsb_internal.h"

namespace gsb {

enum OrthoDtype : int { kOrthoF32 = 0, kOrthoBF16 = 1, kOrthoF16 = 2 };

constexpr int kOrthoMaxSteps = 32;
constexpr int kOrthoMaxTensors = 32; // tensors of one launch
constexpr int kOrthoMaxSide = 2000000000; // rows or columns: sides rounded up to a tile are held in 32 bits

struct OrthoCoefficients {
    int steps;
    float c[kOrthoMaxSteps][3];
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Four values of a type at a 4-value boundary.
template <typename T> struct Quad;
template <> struct Quad<float> {
    using type = float4;
    static __device__ __forceinline__ float4 get(float4 v) { return v; }
    static __device__ __forceinline__ float4 put(float4 f) { return f; }
};
template <> struct Quad<__half> {
    using type = uint2;
    static __device__ __forceinline__ float4 get(uint2 v) {
        const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<__half2 *>(&v.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    static __device__ __forceinline__ uint2 put(float4 f) {
        const __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(f.z, f.w);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};
template <> struct Quad<__nv_bfloat16> {
    using type = uint2;
    static __device__ __forceinline__ float4 get(uint2 v) {
        const float2 a = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v.x)),
                     b = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    static __device__ __forceinline__ uint2 put(float4 f) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
};

// Momentum and the matrix that is orthogonalised, in 32 bits: m <- m + (1 - mu)(g - m),
// u = g + mu (m - g) (Nesterov) or m.
__device__ __forceinline__ float muon_momentum(float g, float m, float one_minus_mu) {
    return fmaf(one_minus_mu, g - m, m);
}
__device__ __forceinline__ float muon_update(float g, float m_new, float mu, int nesterov) {
    return nesterov ? fmaf(mu, m_new - g, g) : m_new;
}
__device__ __forceinline__ float muon_param(float p, float o, float lr, float decay) {
    return fmaf(-lr, o, p * decay);
}

// How a matrix is divided by its norm, a sum in 64 bits: x * pre / div. Where the norm nears the ends of a float's range
// or passes them (FLT_MAX in several entries is a norm above it), a power of two brings it back.
struct Divisor {
    float pre, div;
    bool small; // the norm is below eps, which takes its place
};
__device__ __forceinline__ Divisor divisor_of(double norm, float eps) {
    Divisor d;
    d.small = (float)norm < eps;
    d.pre = d.small ? 1.f : norm > 0x1p120 ? 0x1p-40f : norm < 0x1p-100 ? 0x1p60f : 1.f;
    d.div = d.small ? eps : (float)(norm * (double)d.pre);
    return d;
}

// The tensors of one Muon step that share a shape: [batch_t, rows, cols] each.
// Matrix b of the launch belongs to the tensor t with first[t] <= b < first[t + 1].
struct MuonTable {
    int n;
    int dtype, state_dtype, nesterov;
    float mu, one_minus_mu;
    const bool *valid; // per leading row of every tensor, or NULL
    void *param[kOrthoMaxTensors];
    const void *grad[kOrthoMaxTensors];
    void *momentum[kOrthoMaxTensors];
    float lr[kOrthoMaxTensors], decay[kOrthoMaxTensors]; // decay = 1 - lr * weight_decay
    int inner[kOrthoMaxTensors];         // matrices per leading row
    bool transposed[kOrthoMaxTensors];   // the tensor's matrices are [long, short]
    long long skipped[kOrthoMaxTensors]; // the tensor's matrices before its first one here
    long long first[kOrthoMaxTensors + 1];
};

__device__ __forceinline__ int muon_tensor_of(const MuonTable &t, long long b) {
    int i = 0;
    while (i + 1 < t.n && b >= t.first[i + 1]) ++i;
    return i;
}
__device__ __forceinline__ bool muon_visible(const MuonTable &t, int i, long long b) {
    return t.valid == nullptr || t.valid[(b - t.first[i] + t.skipped[i]) / t.inner[i]];
}

// A launch whose blocks may set up while the launch before it in the stream ends; the kernel
// waits for that one (griddepcontrol.wait) before it touches memory. `cluster` blocks form a cluster.
template <typename... P, typename... A>
inline int launch_clusters_after(void (*kernel)(P...), int cluster, unsigned blocks, int threads, size_t smem, cudaStream_t stream,
                                 const char *what, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return set_error(kErrLaunch, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}
template <typename... P, typename... A>
inline int launch_after(void (*kernel)(P...), unsigned blocks, int threads, size_t smem, cudaStream_t stream, const char *what,
                        const A &...args) {
    return launch_clusters_after(kernel, 0, blocks, threads, smem, stream, what, args...);
}

// --- thin matrices (ortho_thin.cu) -----------------------------------------
// short side <= 4 and long side <= 128: a few lanes hold one matrix.
bool ortho_is_thin(int rows, int cols);
int ortho_thin_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream);
int ortho_thin_bwd(long long batch, int rows, int cols, int dtype, const void *x, const void *v_y, void *v_x,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream);
int ortho_thin_muon(const MuonTable &table, int rows, int cols, const OrthoCoefficients &co, float eps,
                    cudaStream_t stream);

// --- tiled products (ortho_gemm.cu) ----------------------------------------
// A matrix of the iteration: value = scale * (hi + lo), both fp16, so 22
// significand bits. Row-major, rows of `ld` elements (a multiple of 8), one
// matrix after `stride` elements.
struct OrthoPlanes {
    __half *hi, *lo;
    int ld;
    long long stride;
};

// --- short side <= 128 and not too long (ortho_cluster.cu): one launch, the matrix in the
// shared memory of a cluster. The scales are those of X, A and B as OrthoPlanes have them.
int ortho_is_clustered(int rows, int cols); // the blocks of a matrix's cluster, or 0
// Where the first step's X, A and B go for a backward pass (x.hi = NULL: nowhere), each further step's
// `step` halves (2 bytes) behind.
struct ClusterKept {
    OrthoPlanes x, a, b;
    float *da, *db;
    double *norms;
    long long step;
};
int ortho_cluster_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y, const OrthoCoefficients &co,
                      float x_scale, float a_scale, float b_scale, float eps, const ClusterKept &kept, cudaStream_t stream);
// The table's tensors, of sizes[t] = {rows, columns} each, all with the same clusters.
int ortho_cluster_muon(const MuonTable &table, const int sizes[][2], const OrthoCoefficients &co, float x_scale, float a_scale,
                       float b_scale, float eps, cudaStream_t stream);

enum OrthoEpilogue : int {
    kEpiGram,   // A: off-diagonal part and its diagonal
    kEpiSquare, // B from A A
    kEpiApply,  // X <- a X + B X
    kEpiOut,    // the last step, to the caller's tensor
    kEpiMuon,   // the last step, into the parameters
    kEpiSym,    // S = G X^T + X G^T
    kEpiAnti,   // T = b S + c (S A + A S)
};

// C[b] = sum over pairs p of P_p[b] Q_p[b] (M x N, contraction K), then the epilogue,
// with e the element-wise operand, D = diag_in and d = c the constants:
//   kEpiGram    i != j: out = c0 C, i == j: diag_out = c1 C, out = 0
//   kEpiSquare  i != j: out = (c0 + c1 (D_i + D_j)) e + c2 C
//               i == j: diag_out = c3 D + c4 D D + c5 C, out = 0
//   kEpiApply   out = ((c0 + D_i) e + c1 C) c2, kEpiOut and kEpiMuon likewise
//   kEpiSym     out = c0 C
//   kEpiAnti    out = (c0 + c1 (D_i + D_j)) e + c2 C
struct OrthoGemm {
    long long batch;
    int M, N, K;
    int pairs;      // 1 or 2
    int q_k_major;  // Q stored [N, K] (1) or [K, N] (0)
    int symmetric;  // only tiles on and below the diagonal, mirrored when written
    int split;      // products of hi + lo (three products); else of hi alone
    OrthoPlanes p[2], q[2];
    int epilogue;
    float c[6];
    OrthoPlanes e, out;      // the element-wise operand and the result
    const float *diag_in;    // [batch, M]
    float *diag_out;         // [batch, M]
    void *y;                 // kEpiOut: [batch, rows, cols] of `dtype`
    int dtype, transposed;   // transposed: y is [N, M] in memory (kEpiMuon: the table says it)
    int *error;              // set when a kernel's wait ran out; the last product then writes NaN. Where that is the product
                             // whose wait ran out, its block does for all of its tiles
};

int ortho_gemm(const OrthoGemm &g, const MuonTable *table, cudaStream_t stream);

// The tile that a product takes on a GPU of `sms` SMs: its columns (256: of a pair of SMs) and the blocks that share its depth.
struct OrthoTile {
    int columns, ranks;
};
OrthoTile ortho_tile(const OrthoGemm &g, int sms);

} // namespace gsb
