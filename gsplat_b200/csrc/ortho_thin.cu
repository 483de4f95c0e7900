// Thin matrices: the forward pass and what counts as thin.
#include "ortho_thin.cuh"

namespace gsb {

bool ortho_is_thin(int rows, int cols) {
    const int s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    return s <= kThinMaxShort && l <= kThinMaxLong;
}

int ortho_thin_fwd(long long batch, int rows, int cols, int dtype, const void *x, void *y,
                   const OrthoCoefficients &co, float eps, cudaStream_t stream) {
    if (std::max(rows, cols) <= kStackMaxLong) {
        StackShape sk = stack_shape(batch, rows, cols);
        sk.vec = sk.E >= 4 && quads_aligned(x, dtype) && quads_aligned(y, dtype);
        const long long blocks = (batch + kStackThreads - 1) / kStackThreads;
        if (blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "orthogonalize: too many matrices");
        const size_t smem = (size_t)kStackThreads * sk.pitch * sizeof(float);
        return with_type(dtype, [&](auto tv) {
            using T = decltype(tv);
            return with_short(sk.E / sk.L, [&](auto s) {
                return with_rows<kStackMaxLong>(sk.L, [&](auto p) {
                    auto *kernel = stack_fwd_kernel<T, p.value, s.value>;
                    if (!allow_smem(kernel, smem)) return check_launch("stack_fwd_kernel attributes");
                    kernel<<<(unsigned)blocks, kStackThreads, smem, stream>>>(sk, (const T *)x, (T *)y, co, eps);
                    return check_launch("stack_fwd_kernel");
                });
            });
        });
    }
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

} // namespace gsb
