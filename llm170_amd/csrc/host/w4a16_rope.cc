// Norm and rotation of queries and keys (kernels/rope.hip), and the frequencies of the rotation.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "w4a16_internal.h"

extern "C" int w4a16_rope_freqs(size_t rot_dim, double base, int scaling, double factor, double trained, double low, double high, double* freqs, float* amp) {
    if (!freqs || !amp) return w4_fail(W4A16_ERR_ARG, "rope_freqs: null argument");
    if (rot_dim == 0 || rot_dim % 2 != 0 || rot_dim > kW4RopeMaxDim)
        return w4_fail(W4A16_ERR_SHAPE, "rope_freqs: rot_dim=%zu must be even, 2..%d", rot_dim, kW4RopeMaxDim);
    if (scaling < W4A16_ROPE_PLAIN || scaling > W4A16_ROPE_RAMP) return w4_fail(W4A16_ERR_ARG, "rope_freqs: scaling %d (0 = plain, 1 = linear, 2 = bands, 3 = ramp)", scaling);
    const bool scaled = scaling != W4A16_ROPE_PLAIN, bounds = scaling == W4A16_ROPE_BANDS || scaling == W4A16_ROPE_RAMP;
    // negated, so that no NaN passes
    if (!(base > 1.0) || !std::isfinite(base) || (scaled && (!(factor > 0.0) || !std::isfinite(factor))) ||
        (bounds && (!(trained > 0.0) || !std::isfinite(trained) || !(low > 0.0) || !(high > low) || !std::isfinite(high))))
        return w4_fail(W4A16_ERR_ARG, "rope_freqs: base=%g above 1, factor=%g and trained=%g above 0, low=%g above 0 and high=%g above it are needed", base, factor, trained, low, high);
    const double two_pi = 6.283185307179586476925;
    const size_t half = rot_dim / 2;
    double lo = 0.0, hi = 0.0;
    if (scaling == W4A16_ROPE_RAMP) {
        // the pair whose frequency turns so many times within the trained length
        auto pair_of = [&](double turns) { return (double)rot_dim * std::log(trained / (two_pi * turns)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(pair_of(high)), 0.0);
        hi = std::min(std::ceil(pair_of(low)), (double)rot_dim - 1.0);
    }
    for (size_t c = 0; c < half; c++) {
        double f = std::pow(base, -2.0 * (double)c / (double)rot_dim);
        if (scaling == W4A16_ROPE_LINEAR) {
            f /= factor;
        } else if (bounds) {
            // share of the frequency that stays as it was trained
            const double keep = scaling == W4A16_ROPE_BANDS ? (trained * f / two_pi - low) / (high - low) : 1.0 - ((double)c - lo) / std::max(hi - lo, 0.001);
            const double k = std::min(std::max(keep, 0.0), 1.0);
            f *= (1.0 - k) / factor + k;
        }
        freqs[c] = f;
    }
    *amp = scaling == W4A16_ROPE_RAMP && factor > 1.0 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return 0;
}

extern "C" int w4a16_qk_norm_rope(w4a16_ctx* ctx, uint64_t x_dev, int x_type, size_t ldx, size_t t, size_t n_q, size_t n_k, size_t head_dim, uint64_t qw_dev,
                                  uint64_t kw_dev, float eps, uint64_t pos_dev, uint64_t freqs_dev, size_t rot_dim, float amp, int interleaved, uint64_t q_dev,
                                  size_t ldq, uint64_t k_dev, size_t ldk, int y_type) {
    const char* const api = "qk_norm_rope";
    if (!ctx || !x_dev || (n_q && !q_dev) || (n_k && !k_dev)) return w4_fail(W4A16_ERR_ARG, "%s: null operand", api);
    if (!w4_float_type(x_type) || !w4_float_type(y_type)) return w4_fail(W4A16_ERR_ARG, "%s: x type %d, result type %d (0 = f32, 1 = f16, 2 = bf16)", api, x_type, y_type);
    if (t == 0 || t > 0x7fffff00u || n_q > 65536 || n_k > 65536 || n_q + n_k == 0 || head_dim == 0 || head_dim > kW4RopeMaxDim)
        return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu outside 1..2^31-256, n_q=%zu and n_k=%zu up to 65536 and not both 0, head_dim=%zu outside 1..%d", api, t, n_q, n_k,
                       head_dim, kW4RopeMaxDim);
    if (rot_dim % 2 != 0 || rot_dim > head_dim) return w4_fail(W4A16_ERR_SHAPE, "%s: rot_dim=%zu must be even and at most head_dim=%zu", api, rot_dim, head_dim);
    if (rot_dim && (!pos_dev || !freqs_dev)) return w4_fail(W4A16_ERR_ARG, "%s: a rotation needs positions and frequencies", api);
    if (rot_dim == 0 && !qw_dev && !kw_dev) return w4_fail(W4A16_ERR_ARG, "%s: neither a norm nor a rotation is asked for", api);
    if ((qw_dev || kw_dev) && !(eps >= 0.0f)) return w4_fail(W4A16_ERR_ARG, "%s: eps=%g", api, eps);
    const size_t wq = n_q * head_dim, wk = n_k * head_dim;
    if (ldx == 0) ldx = wq + wk;
    if (ldq == 0) ldq = wq;
    if (ldk == 0) ldk = wk;
    if (ldx < wq + wk || ldq < wq || ldk < wk)
        return w4_fail(W4A16_ERR_SHAPE, "%s: ldx=%zu ldq=%zu ldk=%zu below %zu, %zu and %zu columns", api, ldx, ldq, ldk, wq + wk, wq, wk);
    if (x_dev % w4_type_bytes(x_type) || (q_dev | k_dev) % w4_type_bytes(y_type) || (qw_dev | kw_dev | pos_dev) % 4 || freqs_dev % 8)
        return w4_fail(W4A16_ERR_ARG, "%s: operands must be aligned to their elements", api);
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    // pairs per lane: 8 or 2 where both parts of a head are whole units of them, else 1
    const size_t half = rot_dim / 2, rest = head_dim - rot_dim;
    const size_t vec = half % 8 == 0 && rest % 16 == 0 ? 8 : half % 2 == 0 && rest % 4 == 0 ? 2 : 1;
    const size_t units = half / vec + (rest + 2 * vec - 1) / (2 * vec);
    int lg = 0;
    while (lg < 6 && ((size_t)1 << lg) < units) lg++;
    const size_t hp = (size_t)64 >> lg, passes = (n_q + hp - 1) / hp + (n_k + hp - 1) / hp;
    // waves to a row: one pass each while they are fewer than 16 to a CU
    const size_t splits = std::min(passes, std::max<size_t>(1, 16 * (size_t)std::max(ctx->cu_count, 1) / t));
    char sym[64];
    snprintf(sym, sizeof sym, "w4a16_qk_norm_rope_%s_v%zu%s", w4_type_name(x_type), vec, interleaved ? "_il" : "");
    int nq = (int)n_q, nk = (int)n_k, dim = (int)head_dim, rot = (int)rot_dim, sp = (int)splits;
    const size_t most = 0xffffffu * (size_t)4 / splits;  // HIP takes fewer than 2^32 threads in a launch: more rows go in several
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        uint64_t x_at = x_dev + at * ldx * w4_type_bytes(x_type), p_at = pos_dev ? pos_dev + at * 4 : 0, q_at = q_dev + at * ldq * w4_type_bytes(y_type),
                 k_at = k_dev + at * ldk * w4_type_bytes(y_type);
        int ti = (int)rows;
        void* params[] = {&x_at, &ldx, &ti, &nq, &nk, &dim, &rot, &qw_dev, &kw_dev, &eps, &p_at, &freqs_dev, &amp, &q_at, &ldq, &k_at, &ldk, &y_type, &lg, &sp};
        W4_TRY(w4_launch(ctx, sym, (unsigned)((rows * splits + 3) / 4), 1, 256, 0, params));
    }
    return 0;
}
