// Scoring of logits (kernels/score.hip): log probabilities of given tokens, entropy, most likely tokens.
#include <algorithm>

#include "w4a16_internal.h"

// Workgroups per row.  One from 1024 rows on; with fewer a row is cut into segments of whole stages of a workgroup's four waves: about
// 1024 workgroups, but no more than 16 per row, or as many as make 256 workgroups, up to 32 (the records of more cost more than the
// shorter segments save).  us in 1 / 4 / 8 / 16 / 32 segments: 1 x 131072 bf16, 20 best, 35.5 / 21.4 / 16.9 / 14.6 / 14.7; 16 x
// 131072 f32 49.1 / 25.7 / 20.0 / 18.2 / 21.1; 64 x 131072 bf16 41.4 / 23.9 / 20.9 / 20.7 / -; 256 x 131072 f16 39.2 / 31.6 / 36.8 / 49.0;
// 600 x 100003 f16, 5 best, 41.5 / 50.3 / 48.2 / 64.7; 1000 x 32000 bf16 28.5 / 54.0.
static size_t score_segments(size_t t, size_t vocab, size_t cus, size_t stage) {
    const size_t most = (vocab + stage - 1) / stage, few = std::max(cus / t, std::min<size_t>(4 * cus / t, 16));
    return std::max<size_t>(1, std::min({most, few, (size_t)32}));
}

extern "C" int w4a16_token_logprobs(w4a16_ctx* ctx, uint64_t logits_dev, int logits_type, size_t ld, size_t t, size_t n_vocab,
                                    uint64_t targets_dev, uint64_t logp_dev, uint64_t entropy_dev, size_t top_k, uint64_t top_idx_dev,
                                    uint64_t top_logp_dev) {
    if (!ctx || !logits_dev) return w4_fail(W4A16_ERR_ARG, "token_logprobs: null operand");
    if (logits_type != W4A16_F32 && logits_type != W4A16_F16 && logits_type != W4A16_BF16)
        return w4_fail(W4A16_ERR_ARG, "token_logprobs: logits type %d (0 = f32, 1 = f16, 2 = bf16)", logits_type);
    if (t == 0 || t > 0x7fffff00u || n_vocab == 0 || n_vocab > 0x7fffff00u)
        return w4_fail(W4A16_ERR_SHAPE, "token_logprobs: t=%zu n_vocab=%zu outside 1..2^31-256", t, n_vocab);
    if (ld == 0) ld = n_vocab;
    if (ld < n_vocab) return w4_fail(W4A16_ERR_SHAPE, "token_logprobs: ld=%zu below n_vocab=%zu", ld, n_vocab);
    if (top_k > kW4ScoreMaxTop || top_k > n_vocab)
        return w4_fail(W4A16_ERR_SHAPE, "token_logprobs: top_k=%zu above %d or n_vocab=%zu", top_k, kW4ScoreMaxTop, n_vocab);
    if ((logp_dev != 0) != (targets_dev != 0)) return w4_fail(W4A16_ERR_ARG, "token_logprobs: targets and logp come together");
    if (top_k ? !top_idx_dev && !top_logp_dev : top_idx_dev || top_logp_dev)
        return w4_fail(W4A16_ERR_ARG, "token_logprobs: top_k=%zu and its results come together", top_k);
    if (!logp_dev && !entropy_dev && !top_k) return w4_fail(W4A16_ERR_ARG, "token_logprobs: no result asked for");
    if (logits_dev % (logits_type == W4A16_F32 ? 4 : 2) || (targets_dev | logp_dev | entropy_dev | top_idx_dev | top_logp_dev) % 4)
        return w4_fail(W4A16_ERR_ARG, "token_logprobs: operands must be aligned to their elements");
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    const size_t stage = kW4ScoreStageBytes * 4 / (logits_type == W4A16_F32 ? 4 : 2);
    const size_t want = score_segments(t, n_vocab, (size_t)std::max(ctx->cu_count, 1), stage);
    const size_t seg_len = ((n_vocab + want - 1) / want + stage - 1) / stage * stage, segs = (n_vocab + seg_len - 1) / seg_len;
    if (segs > 1) {
        W4_TRY(w4_ensure(ctx, &ctx->score_ws, &ctx->score_ws_cap, t * segs * kW4ScoreRecord));
        if (t * 4 > ctx->score_tickets_cap) {
            W4_TRY(w4_ensure(ctx, &ctx->score_tickets, &ctx->score_tickets_cap, std::max<size_t>(t * 4, 8192)));
            const int rc = w4a16_memset0(ctx, ctx->score_tickets, ctx->score_tickets_cap);
            if (rc) ctx->score_tickets_cap = 0;  // not cleared: asked for anew
            W4_TRY(rc);
        }
    }
    uint64_t ws = ctx->score_ws, tickets = ctx->score_tickets;
    int v = (int)n_vocab, top = (int)top_k, sg = (int)segs, sl = (int)std::min<size_t>(seg_len, 0x7fffffff);
    const char* sym = logits_type == W4A16_F32 ? "w4a16_token_logprobs_f32" : logits_type == W4A16_F16 ? "w4a16_token_logprobs_f16" : "w4a16_token_logprobs_bf16";
    // HIP takes fewer than 2^32 threads in a launch: more rows go in several.  Rows in segments are fewer than 1024.
    const size_t most = 0xffffffu;
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        auto from = [&](uint64_t p, size_t bytes) { return p ? p + at * bytes : 0; };
        uint64_t z = logits_dev + at * ld * (logits_type == W4A16_F32 ? 4 : 2), tg = from(targets_dev, 4), lp = from(logp_dev, 4), en = from(entropy_dev, 4),
                 ti = from(top_idx_dev, top_k * 4), tl = from(top_logp_dev, top_k * 4);
        void* params[] = {&z, &ld, &v, &tg, &lp, &en, &top, &ti, &tl, &sg, &sl, &ws, &tickets};
        W4_TRY(w4_launch(ctx, sym, (unsigned)(rows * segs), 1, 256, 0, params));
    }
    return 0;
}
