// C-ABI entry points of the gated feed-forward product (include/flint/flint_gated.h):
// a Checker chain and the launches of the GEMM kernels.
#include "common/args.h"
#include "flint/flint_gated.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::Span;

Checker& gated_sizes(Checker& c, size_t m, size_t n, size_t k, int activation) {
    return c
        .require(activation == FLINT_GATE_SILU || activation == FLINT_GATE_GELU,
                 "activation (%d) must be 0 or 1", activation)
        .require(k != 0 && k % 8 == 0, "k (%zu) must be a positive multiple of 8", k)
        .require(n % 8 == 0, "n (%zu) must be a multiple of 8", n)
        .require(m <= flint::kGemmMaxMN && n <= flint::kGemmMaxMN / 2 && k <= flint::kGemmMaxK &&
                     m <= flint::kGatedMaxOutputs / n,
                 "%zu x %zu x %zu is too large: m can be up to %zu, n up to %zu, m n up to %zu, and "
                 "k up to %zu",
                 m, n, k, flint::kGemmMaxMN, flint::kGemmMaxMN / 2, flint::kGatedMaxOutputs,
                 flint::kGemmMaxK);
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_gemm_nt_gated(void* y, void* pre, const void* x, const void* w,
                                           const void* bias, size_t m, size_t n, size_t k,
                                           int activation, flint_stream stream) {
    if (m == 0 || n == 0) return FLINT_OK;
    Checker c("flint_gemm_nt_gated");
    if (!gated_sizes(c, m, n, k, activation).ok()) return c.status();
    const Span sy{"y", y, m * n * 2}, sx{"x", x, m * k * 2}, sw{"w", w, 2 * n * k * 2};
    const Span sp{"pre", pre, 2 * m * n * 2}, sb{"bias", bias, 2 * n * 4};
    c.operands({sy, sx, sw}).apart(sy, {sx, sw});
    if (bias != nullptr) c.operands({sb}).apart(sy, {sb});
    if (pre != nullptr) {
        c.operands({sp}).apart(sp, {sy, sx, sw});
        if (bias != nullptr) c.apart(sp, {sb});
    }
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_gemm_nt_gated(y, pre, x, w, bias, activation == FLINT_GATE_GELU, m,
                                                n, k, flint::to_hip(stream)));
    return FLINT_OK;
}

FLINT_API flint_status flint_gemm_nn_dgated(void* dpre, const void* x, const void* w,
                                            const void* pre, size_t m, size_t n, size_t k,
                                            int activation, flint_stream stream) {
    if (m == 0 || n == 0) return FLINT_OK;
    Checker c("flint_gemm_nn_dgated");
    if (!gated_sizes(c, m, n, k, activation).ok()) return c.status();
    const Span out{"dpre", dpre, 2 * m * n * 2}, sx{"x", x, m * k * 2}, sw{"w", w, n * k * 2},
        sp{"pre", pre, 2 * m * n * 2};
    if (!c.operands({out, sx, sw, sp}).apart(out, {sx, sw, sp}).ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_gemm_nn_dgated(dpre, x, w, pre, activation == FLINT_GATE_GELU, m, n,
                                                 k, flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
