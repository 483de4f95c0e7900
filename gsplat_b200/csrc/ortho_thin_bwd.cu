// Thin matrices: the backward pass.
#include "ortho_thin.cuh"

namespace gsb {

int ortho_thin_bwd(long long batch, int rows, int cols, int dtype, const void *x, const void *v_y, void *v_x,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream) {
    if (std::max(rows, cols) <= kStackMaxLongBwd) {
        StackShape sk = stack_shape(batch, rows, cols);
        sk.vec = sk.E >= 4 && quads_aligned(x, dtype) && quads_aligned(v_y, dtype) && quads_aligned(v_x, dtype);
        const int S = sk.E / sk.L, R = sk.L <= 4 ? 4 : sk.L <= 8 ? 8 : 16;
        for (int threads = kStackThreads; threads >= 64; threads /= 2) { // many steps of many rows: the grouped kernel
            const size_t smem = (((size_t)threads * sk.pitch + 1) / 2 * 2 + (size_t)co.steps * R * S * threads) * sizeof(float);
            if (smem > kStackSmem) continue;
            const long long blocks = (batch + threads - 1) / threads;
            if (blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "orthogonalize: too many matrices");
            return with_type(dtype, [&](auto tv) {
                using T = decltype(tv);
                return with_short(S, [&](auto s) {
                    return with_rows<kStackMaxLongBwd>(sk.L, [&](auto p) {
                        auto *kernel = stack_bwd_kernel<T, p.value, s.value>;
                        if (!allow_smem(kernel, smem)) return check_launch("stack_bwd_kernel attributes");
                        kernel<<<(unsigned)blocks, threads, smem, stream>>>(sk, (const T *)x, (const T *)v_y, (T *)v_x, co, eps);
                        return check_launch("stack_bwd_kernel");
                    });
                });
            });
        }
    }
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

} // namespace gsb
