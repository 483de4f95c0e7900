// Thin matrices: the Muon step.
#include "ortho_thin.cuh"

namespace gsb {

int ortho_thin_muon(const MuonTable &table, int rows, int cols, const OrthoCoefficients &co, float eps,
                    cudaStream_t stream) {
    if (std::max(rows, cols) <= kStackMaxLong) {
        const StackShape sk = stack_shape(table.first[table.n], rows, cols);
        StackBlocks sb = {};
        // with a mask, as many turns a block as leave each SM a few blocks and their stages fit three times
        sb.span = kStackThreads;
        while (table.valid != nullptr && sb.span < kStackSpan && sk.batch / (2 * sb.span) >= 4 * 148 &&
               2 * sb.span * sk.pitch * sizeof(float) <= 48 * 1024)
            sb.span *= 2;
        for (int i = 0; i < table.n; ++i) {
            sb.first[i + 1] = sb.first[i] + (table.first[i + 1] - table.first[i] + sb.span - 1) / sb.span;
            sb.vec[i] = sk.E >= 4 && quads_aligned(table.param[i], table.dtype) && quads_aligned(table.grad[i], table.dtype) &&
                        quads_aligned(table.momentum[i], table.state_dtype);
        }
        const long long blocks = sb.first[table.n];
        if (blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "muon: too many matrices");
        const size_t smem = ((size_t)sb.span * sk.pitch + 4) * sizeof(float); // a last quad may be read past its matrix
        return with_type(table.dtype, [&](auto tv) {
            using T = decltype(tv);
            return with_short(sk.E / sk.L, [&](auto s) {
                return with_rows<kStackMaxLong>(sk.L, [&](auto p) {
                    auto launch = [&](auto *kernel) {
                        if (!allow_smem(kernel, smem)) return check_launch("stack_muon_kernel attributes");
                        kernel<<<(unsigned)blocks, kStackThreads, smem, stream>>>(sk, table, sb, co, eps);
                        return check_launch("stack_muon_kernel");
                    };
                    return table.state_dtype == table.dtype ? launch(stack_muon_kernel<T, T, p.value, s.value>)
                                                            : launch(stack_muon_kernel<T, float, p.value, s.value>);
                });
            });
        });
    }
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
