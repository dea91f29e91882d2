// Verification of drafted tokens (kernels/verify.hip).
#include <algorithm>
#include <cstdio>

#include "w4a16_internal.h"

extern "C" int w4a16_verify_drafts(w4a16_ctx* ctx, uint64_t logits_dev, int logits_type, size_t ld, uint64_t draft_dev, size_t ld_draft, size_t t, size_t n_vocab,
                                   uint64_t row0_dev, size_t seqs, uint64_t drafted_dev, uint64_t u_dev, uint64_t temps_dev, uint64_t tokens_dev, uint64_t accepted_dev) {
    const char* const api = "verify_drafts";
    if (!ctx || !logits_dev || !row0_dev || !drafted_dev || !u_dev || !tokens_dev || !accepted_dev) return w4_fail(W4A16_ERR_ARG, "%s: null operand", api);
    if (!w4_float_type(logits_type)) return w4_fail(W4A16_ERR_ARG, "%s: logits type %d (0 = f32, 1 = f16, 2 = bf16)", api, logits_type);
    if (t == 0 || t > 0x3fffffffu || seqs == 0 || seqs > 0x3fffffffu || n_vocab == 0 || n_vocab > 0x3fffffffu)
        return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu seqs=%zu n_vocab=%zu outside 1..2^30-1", api, t, seqs, n_vocab);
    if (ld == 0) ld = n_vocab;
    if (ld_draft == 0) ld_draft = n_vocab;
    if (ld < n_vocab || ld_draft < n_vocab) return w4_fail(W4A16_ERR_SHAPE, "%s: ld=%zu, ld_draft=%zu below n_vocab=%zu", api, ld, ld_draft, n_vocab);
    if ((logits_dev | draft_dev) % w4_type_bytes(logits_type) || (row0_dev | drafted_dev | u_dev | temps_dev | tokens_dev | accepted_dev) % 4)
        return w4_fail(W4A16_ERR_ARG, "%s: operands must be aligned to their elements", api);
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    // Elements of a segment, of whole stages of a workgroup's four waves.  Rows: as many segments as make twelve workgroups to a CU; us with 1 / 4 / 8 / 12 / 16 / 24 / 40 of them: 193 rows
    // of 131072 bf16 with drafts 24.0 / 21.3 / 22.9 / 22.4 / 25.2 / 25.7 / 37.5; 400 of 100003 f16 41.0 / 40.8 / 40.7 / 32.4 / 31.1 / 33.3 / 33.5.  Pick: one stage.
    const size_t stage = 4 * 4096 / w4_type_bytes(logits_type), streams = draft_dev ? 2 : 1, cus = (size_t)std::max(ctx->cu_count, 1);
    const size_t stages = (n_vocab + stage - 1) / stage, want = std::min(stages, std::max<size_t>(1, 12 * cus / (t * streams)));
    const size_t seg = (stages + want - 1) / want * stage, segs = (n_vocab + seg - 1) / seg;
    const size_t pick_segs = stages;
    if (pick_segs > 0xffffffu / streams || t * streams > 0xffffffffffu / segs || seqs > 0xffffffffffu / pick_segs)
        return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu seqs=%zu n_vocab=%zu exceed the scratch", api, t, seqs, n_vocab);
    const size_t rows_at = t * streams * segs * 16, parts_at = rows_at + t * 32, bytes = parts_at + seqs * pick_segs * 4 * 40;  // a part of a row to each wave
    W4_TRY(w4_ensure(ctx, &ctx->verify_ws, &ctx->verify_ws_cap, bytes));
    if ((t + seqs) * 4 > ctx->verify_tickets_cap) {
        W4_TRY(w4_ensure(ctx, &ctx->verify_tickets, &ctx->verify_tickets_cap, std::max<size_t>((t + seqs) * 4, 8192)));
        const int rc = w4a16_memset0(ctx, ctx->verify_tickets, ctx->verify_tickets_cap);
        if (rc) ctx->verify_tickets_cap = 0;  // not cleared: asked for anew
        W4_TRY(rc);
    }
    uint64_t sums = ctx->verify_ws, rows = sums + rows_at, parts = sums + parts_at, row_tickets = ctx->verify_tickets, seq_tickets = row_tickets + t * 4;
    int v = (int)n_vocab, ti = (int)t, nb = (int)seqs, sg = (int)segs, sl = (int)std::min<size_t>(seg, 0x7fffffff), psg = (int)pick_segs, first = 0;
    char sym[64];
    // HIP takes fewer than 2^32 threads in a launch: more rows or sequences go in several
    snprintf(sym, sizeof sym, "w4a16_verify_rows_%s", w4_type_name(logits_type));
    const size_t per_row = streams * segs, most_rows = 0xffffffu / per_row, most_seqs = 0xffffffu / pick_segs;
    for (size_t at = 0; at < t; at += most_rows) {
        first = (int)at;
        void* params[] = {&logits_dev, &ld, &draft_dev, &ld_draft, &v, &ti, &first, &row0_dev, &nb, &drafted_dev, &u_dev, &temps_dev, &sg, &sl, &sums, &rows, &row_tickets};
        W4_TRY(w4_launch(ctx, sym, (unsigned)(std::min(most_rows, t - at) * per_row), 1, 256, 0, params));
    }
    snprintf(sym, sizeof sym, "w4a16_verify_pick_%s", w4_type_name(logits_type));
    for (size_t at = 0; at < seqs; at += most_seqs) {
        first = (int)at;
        void* params[] = {&logits_dev, &ld, &draft_dev, &ld_draft, &v, &ti, &first, &row0_dev, &drafted_dev, &u_dev, &temps_dev, &psg, &rows, &parts, &seq_tickets,
                          &tokens_dev, &accepted_dev};
        W4_TRY(w4_launch(ctx, sym, (unsigned)(std::min(most_seqs, seqs - at) * pick_segs), 1, 256, 0, params));
    }
    return 0;
}
