// W8A8 linears: registration, quantisation of activation rows, regime dispatch (kernels/quant.hip, kernels/w8a8.hip).
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <memory>
#include <new>

#include "w4a16_internal.h"

static inline unsigned ceil_div(size_t a, size_t b) { return (unsigned)((a + b - 1) / b); }

static size_t k_tiles(size_t k) { return w4_q8_blocks(k) * 2; }

int w4_q8_check_rows(const char* what, size_t t, size_t k) {
    if (t == 0 || t > 0x7fffff00u || k == 0 || k > kW4Q8MaxK)
        return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu k=%zu outside 1..2^31-256 and 1..%d", what, t, k, kW4Q8MaxK);
    return 0;
}

extern "C" size_t w4a16_q8_bytes(size_t t, size_t k) {
    if (t == 0 || t > 0x7fffff00u || k == 0 || k > kW4Q8MaxK) return 0;
    const size_t r = w4_q8_tile_rows(t);
    return (t + r - 1) / r * r * k_tiles(k) * 64;
}

static int quant_rows(w4a16_ctx* ctx, uint64_t x, int x_type, size_t ldx, size_t t, size_t k, uint64_t q, uint64_t s) {
    char sym[64];
    // Few rows: a thread per four columns; else one per sixteen, of at most 768 (300 x 17408 f16 10.7 us with 1024, 8.7; 4096 rows 64 and 52)
    const bool few = t <= 16;
    snprintf(sym, sizeof sym, "w4a16_quant_%s_%s", few ? "few" : "rows", w4_type_name(x_type));
    const int r = (int)w4_q8_tile_rows(t);
    const unsigned block = (unsigned)std::min<size_t>(few ? (k + 255) / 256 * 64 : (k + 1023) / 1024 * 64, few ? 1024 : 768);
    int ki = (int)k, kt = (int)k_tiles(k), ri = r, bi = (int)block;
    const size_t most = w4_rows_per_launch(block);
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        uint64_t x_at = x + at * ldx * w4_type_bytes(x_type), q_at = q + at * kt * 64, s_at = s + at * 4;
        int ti = (int)rows;
        void* params[] = {&x_at, &ldx, &ki, &kt, &ri, &q_at, &s_at, &ti, &bi};
        W4_TRY(w4_launch(ctx, sym, few ? (unsigned)rows : ceil_div(rows, 128) * 128, few ? ceil_div(k, block * 4) : 1, block, 0, params));
    }
    return 0;
}

extern "C" int w4a16_quant_rows(w4a16_ctx* ctx, uint64_t x_dev, int x_type, size_t ldx, size_t t, size_t k, uint64_t q_dev, uint64_t s_dev) {
    if (!ctx || !x_dev || !q_dev || !s_dev) return w4_fail(W4A16_ERR_ARG, "quant_rows: null operand");
    if (!w4_float_type(x_type)) return w4_fail(W4A16_ERR_ARG, "quant_rows: x type %d (0 = f32, 1 = f16, 2 = bf16)", x_type);
    W4_TRY(w4_q8_check_rows("quant_rows", t, k));
    if (ldx == 0) ldx = k;
    if (ldx < k) return w4_fail(W4A16_ERR_SHAPE, "quant_rows: ldx=%zu below k=%zu", ldx, k);
    if (x_dev % w4_type_bytes(x_type) || s_dev % 4 || q_dev % 16)
        return w4_fail(W4A16_ERR_ARG, "quant_rows: x and s must be aligned to their elements, q to 16 bytes");
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    return quant_rows(ctx, x_dev, x_type, ldx, t, k, q_dev, s_dev);
}

extern "C" int w4a16_norm_resid_q8(w4a16_ctx* ctx, uint64_t x_dev, uint64_t nw_dev, uint64_t ab_dev, uint64_t q_dev, uint64_t s_dev, size_t t,
                                   size_t w_off, size_t hidden) {
    if (!ctx || !x_dev || !nw_dev || !ab_dev || !q_dev || !s_dev) return w4_fail(W4A16_ERR_ARG, "norm_resid_q8: null operand");
    if (hidden == 0 || hidden > 8192) return w4_fail(W4A16_ERR_SHAPE, "norm_resid_q8: hidden=%zu outside 1..8192", hidden);
    if (w_off > 0x7fffffffu - hidden) return w4_fail(W4A16_ERR_SHAPE, "norm_resid_q8: w_off=%zu too large", w_off);
    W4_TRY(w4_q8_check_rows("norm_resid_q8", t, hidden));
    if (x_dev % 4 || nw_dev % 4 || ab_dev % 4 || s_dev % 4 || q_dev % 16)
        return w4_fail(W4A16_ERR_ARG, "norm_resid_q8: f32 operands must be aligned to 4 bytes, q to 16");
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    int wo = (int)w_off, h = (int)hidden, kt = (int)k_tiles(hidden), r = (int)w4_q8_tile_rows(t);
    const size_t most = w4_rows_per_launch(1024);
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        uint64_t x_at = x_dev + at * hidden * 4, ab_at = ab_dev + at * hidden * 4, q_at = q_dev + at * kt * 64, s_at = s_dev + at * 4;
        int ti = (int)rows;
        void* params[] = {&x_at, &nw_dev, &ab_at, &q_at, &s_at, &wo, &h, &kt, &r, &ti};
        W4_TRY(w4_launch(ctx, "w4a16_norm_resid_q8", r == 16 ? ceil_div(rows, 128) * 128 : (unsigned)rows, 1, 1024, 0, params));
    }
    return 0;
}

// ------------------------------------------------------------------------------------------------ registration
static void free_w8(w4a16_ctx* ctx, W8Lin& L) {
    (void)w4a16_free(ctx, L.q);
    (void)w4a16_free(ctx, L.s);
    L = W8Lin();
}

static float w4_f16_to_f32(uint16_t h) {
    const float sign = h & 0x8000u ? -1.0f : 1.0f;
    const int exp = (h >> 10) & 0x1f, frac = h & 0x3ff;
    if (exp == 0x1f) return frac ? NAN : sign * INFINITY;
    return sign * (exp ? std::ldexp((float)(1024 + frac), exp - 25) : std::ldexp((float)frac, -24));
}

float w4_scale_at(const void* s, int type, size_t i) {
    uint32_t b = 0;
    if (type == W4A16_F32) {
        memcpy(&b, static_cast<const char*>(s) + i * 4, 4);
    } else {
        uint16_t h;
        memcpy(&h, static_cast<const char*>(s) + i * 2, 2);
        if (type == W4A16_F16) return w4_f16_to_f32(h);
        b = (uint32_t)h << 16;
    }
    float v;
    memcpy(&v, &b, 4);
    return v;
}

extern "C" int w4a16_upload_lin_w8a8(w4a16_ctx* ctx, const char* name, const void* q, size_t qlen_bytes, const void* s, size_t slen_bytes, size_t n,
                                     size_t k, int s_type) {
    if (!ctx || !name || !q || !s) return w4_fail(W4A16_ERR_ARG, "upload_lin_w8a8: null argument");
    if (!w4_float_type(s_type)) return w4_fail(W4A16_ERR_ARG, "upload_lin_w8a8 %s: scale type %d (0 = f32, 1 = f16, 2 = bf16)", name, s_type);
    if (n == 0 || n > 0x7fffff00u || k == 0 || k > kW4Q8MaxK || qlen_bytes != n * k || slen_bytes != n * w4_type_bytes(s_type))
        return w4_fail(W4A16_ERR_SHAPE, "upload_lin_w8a8 %s: q=%zu s=%zu bytes for n=%zu k=%zu (k up to %d)", name, qlen_bytes, slen_bytes, n, k,
                       kW4Q8MaxK);
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    W8Lin L;
    L.n = n;
    L.k = k;
    const size_t row_blocks = (n + 15) / 16, kt = k_tiles(k), chunks = row_blocks * kt * 64;
    std::unique_ptr<float[]> scales(new (std::nothrow) float[row_blocks * 16]());
    if (!scales) return w4_fail(W4A16_ERR_ARG, "upload_lin_w8a8 %s: no host memory for %zu scales", name, n);
    for (size_t i = 0; i < n; i++) scales[i] = w4_scale_at(s, s_type, i);
    uint64_t raw = 0;
    int rc = w4a16_alloc(ctx, chunks * 16, &L.q);
    if (!rc) rc = w4a16_alloc(ctx, row_blocks * 64, &L.s);
    if (!rc) rc = w4a16_alloc(ctx, qlen_bytes, &raw);
    if (!rc) rc = w4a16_h2d(ctx, raw, q, qlen_bytes);
    if (!rc) rc = w4a16_h2d(ctx, L.s, scales.get(), row_blocks * 64);
    if (!rc) {
        size_t ns = n, cs = chunks;
        int ki = (int)k, kti = (int)kt;
        void* params[] = {&raw, &L.q, &ns, &ki, &kti, &cs};
        rc = w4_launch(ctx, "w4a16_tile_w8", std::min<unsigned>(ceil_div(chunks, 256), 65536), 1, 256, 0, params);
    }
    if (!rc) rc = w4a16_sync(ctx);
    const std::string keep = rc ? w4_err_save() : std::string();
    (void)w4a16_free(ctx, raw);
    if (rc) {
        free_w8(ctx, L);
        w4_err_restore(keep);
        return rc;
    }
    auto it = ctx->w8lins.find(std::string_view(name));
    if (it != ctx->w8lins.end()) {
        free_w8(ctx, it->second);
        ctx->scratch_gen++;  // graphs captured so far hold the old weights' address
        it->second = L;
    } else {
        ctx->w8lins.emplace(name, L);
    }
    return 0;
}

static int find_w8(w4a16_ctx* ctx, const char* name, const W8Lin** out) {
    if (!ctx || !name) return w4_fail(W4A16_ERR_ARG, "lin_w8a8: null argument");
    auto it = ctx->w8lins.find(std::string_view(name));
    if (it == ctx->w8lins.end()) return w4_fail(W4A16_ERR_NOT_FOUND, "lin_w8a8 %s: not registered", name);
    *out = &it->second;
    return 0;
}

extern "C" int w4a16_lin_w8a8_info(w4a16_ctx* ctx, const char* name, size_t* n, size_t* k) {
    const W8Lin* L = nullptr;
    W4_TRY(find_w8(ctx, name, &L));
    if (n) *n = L->n;
    if (k) *k = L->k;
    return 0;
}

// ------------------------------------------------------------------------------------------------ forward
// Launch of the kernel for groups of up to 64 rows: row blocks per workgroup, waves, k slices; a function of the shape alone.
struct SkinnyPlan {
    int rb = 1, waves = 8, nks = 1;
    double price = 0.0;
};

static SkinnyPlan plan_skinny(size_t n, size_t k, size_t t, size_t cus, bool glu) {
    const size_t kt = k_tiles(k), blocks16 = (n + 15) / 16;
    const size_t groups = (t + 63) / 64;
    const int tt = (int)((t + 16 * groups - 1) / (16 * groups));
    SkinnyPlan best;
    best.price = 1e30;
    for (int rb = 4; rb >= (glu ? 2 : 1); rb /= 2) {
        for (int nks = 1; nks <= 8; nks++) {
            const size_t blocks = (blocks16 + rb - 1) / rb, grid = blocks * nks * groups;
            if (nks > 1 && ((size_t)nks * 8 > kt || grid > 4 * cus)) break;
            const double run = (double)kt / nks;
            // Price in us, fitted to 3000 launches of 19 shapes (n 512 .. 65536, k 1024 .. 17408) at 1 .. 64 rows, cold weights: what it
            // picks is 1.7 % slower in the mean than the best of them.  A CU takes 50 KiB per us of weights and half of the activations'
            // (from the L2); workgroups over those that all CUs have cost nearly a whole one; slices cost a hand-over and their sums' way
            // through memory.  5120 x 17408 at t = 16: one row block, whole k 23.9 us, four and three slices 17.7; 7168 x 5120 at t = 64:
            // 17.5, two row blocks 12.7.  Several groups have the weights from the L2, too: fitted, with the launch itself, to 1100 launches
            // of 19 shapes (n 64 .. 34816, k 320 .. 17408) at 65 .. 600 rows.
            const size_t full = grid / cus, rest = grid % cus;
            const double rounds = (double)full + (rest == 0 ? 0.0 : full == 0 ? 1.0 : 0.94 + 0.06 * (double)rest / (double)cus);
            const double load = run * (rb + (groups > 1 ? 0.28 : 0.48) * (t <= 4 ? 0.25 : tt));
            const double sums = 1e-6 * nks * n * t * 8, join = nks == 1 ? 0.0 : groups > 1 ? 0.91 + 0.37 * sums : 2.07 + 0.24 * sums;
            SkinnyPlan p;
            p.rb = rb;
            p.nks = nks;
            // four waves where a CU has several workgroups and eight would have few k tiles each or hold many sums, or k is short
            p.waves = (grid > cus && (run <= 40 || rb * tt >= 16)) || run <= 16 ? 4 : 8;
            p.waves = (int)std::min<size_t>(p.waves, kt);  // kt is 2 at least, and so are they
            p.price = (groups > 1 ? 4.3 : 0.0) + std::max(rounds * load / (groups > 1 ? 34.2 : 49.6), (double)(blocks16 * kt) / 9079.0) + join;
            if (p.price < best.price) best = p;
        }
    }
    return best;
}

int w4_split_workspace(w4a16_ctx* ctx, size_t part_bytes, size_t tickets) {
    W4_TRY(w4_ensure(ctx, &ctx->w8_part, &ctx->w8_part_cap, part_bytes));
    if (tickets * 4 > ctx->w8_tickets_cap) {
        W4_TRY(w4_ensure(ctx, &ctx->w8_tickets, &ctx->w8_tickets_cap, std::max<size_t>(tickets * 4, 16384)));
        const int rc = w4a16_memset0(ctx, ctx->w8_tickets, ctx->w8_tickets_cap);
        if (rc) ctx->w8_tickets_cap = 0;  // not cleared: asked for anew
        W4_TRY(rc);
    }
    return 0;
}

// Launch of the tiled kernel: rows and columns (of weights) per tile, k slices; a function of the shape alone.
struct TiledPlan {
    int bm = 64, bn = 128, nks = 1;
    double price = 0.0;
};

static TiledPlan plan_tiled(size_t n, size_t k, size_t t, size_t cus) {
    // Price in us, fitted to 1100 launches of 15 shapes (n 688 .. 34816, k 320 .. 17408) at 65 .. 2048 rows, cold weights: what it and the
    // price above pick is 1.6 % slower in the mean than the best of both.  us per k tile of a workgroup alone on its CU and of as many as
    // a CU holds; a round over those costs between its share and a whole one; slices cost their sums' way through memory.  The best by
    // tile: 16000 x 2048 at t = 128 64 x 128 11.8 us, 64 x 256 15.2, 128 x 256 17.9; 5120 x 17408 at t = 300 48.2 in two slices, 49.4 in
    // two, 44.0 in four; 22016 x 4096 gated at t = 1000 123, 113, 91.  Against groups of 64 rows: 64 x 8256 at t = 256 groups
    // 6.4 us, tiles 12; 4096 x 4096 at t = 128 10.0 and 10.8, at t = 400 19.5 and 15; 34816 x 5120 gated at t = 100 72 and 52.
    static const struct { int bm, bn, per_cu; double alone, full; } kTiles[] = {{64, 128, 3, 0.18, 0.50}, {64, 256, 2, 0.29, 0.57}, {128, 256, 2, 0.42, 0.90}};
    const size_t kt = k_tiles(k);
    TiledPlan best;
    best.price = 1e30;
    for (const auto& T : kTiles) {
        for (int nks = 1; nks <= 8; nks++) {
            const size_t grid = (t + T.bm - 1) / T.bm * ((n + T.bn - 1) / T.bn) * nks;
            if (nks > 1 && ((size_t)nks * 8 > kt || grid > T.per_cu * cus)) break;
            const double load = (double)grid / (double)cus, rounds = load / T.per_cu;
            const double per_k = rounds <= 1.0 ? T.alone + (T.full - T.alone) * (std::ceil(load) - 1.0) / (T.per_cu - 1)
                                               : T.full * (0.5 * std::ceil(rounds) + 0.5 * rounds);
            TiledPlan p;
            p.bm = T.bm;
            p.bn = T.bn;
            p.nks = nks;
            p.price = 4.7 + (double)((kt + nks - 1) / nks) * per_k + (nks > 1 ? (nks + 8.5 * load) * T.bm * T.bn / 32768.0 : 0.0);
            if (p.price < best.price) best = p;
        }
    }
    return best;
}

// The kernel that t rows through a linear go to, its grid, and the scratch of its k slices
struct W8Launch {
    char kernel[64] = "";
    size_t grid_x = 0, grid_y = 1, tickets = 0, part_bytes = 0;
    int block = 256, nks = 1, band = 0;  // band: tile rows of a band, 0 = the kernel for groups of up to 64 rows
};

static int plan_w8a8(const char* what, size_t n, size_t k, size_t t, size_t cus, bool glu, W8Launch* out) {
    W8Launch& P = *out;
    const SkinnyPlan few = plan_skinny(n, k, t, cus, glu);
    const TiledPlan tiles = t <= 64 ? TiledPlan() : plan_tiled(n, k, t, cus);
    if (t <= 64 || (t <= 1024 && few.price < tiles.price)) {
        const size_t groups = (t + 63) / 64;  // of as many rows each as can be
        const int tt = (int)((t + 16 * groups - 1) / (16 * groups));
        const size_t blocks16 = (n + 15) / 16;
        snprintf(P.kernel, sizeof P.kernel, "w4a16_w8a8_skinny_r%d_t%d%s", few.rb, tt, glu ? "_glu" : "");
        P.nks = few.nks;
        P.grid_x = glu ? ceil_div(blocks16 / 2, few.rb / 2) : ceil_div(blocks16, few.rb);
        P.grid_y = few.nks * groups;
        P.block = few.waves * 64;
        P.tickets = P.grid_x * groups;
        P.part_bytes = P.tickets * few.nks * few.rb * tt * 1024;
    } else {
        snprintf(P.kernel, sizeof P.kernel, "w4a16_w8a8_tiled_m%d%s%s", tiles.bm, tiles.bn == 128 ? "_n128" : "", glu ? "_glu" : "");
        P.nks = tiles.nks;
        P.tickets = (t + tiles.bm - 1) / tiles.bm * ((n + tiles.bn - 1) / tiles.bn);
        P.part_bytes = P.tickets * tiles.nks * tiles.bm * tiles.bn * 4;
        P.grid_x = (P.tickets * tiles.nks + 7) / 8 * 8;
        // 1024 rows of tiles share their weights in the L2: 34816 x 5120 gated at t = 4096 673 us in an earlier state, 512 rows 679, 256 rows 727
        P.band = 1024 / tiles.bm;
    }
    if (P.grid_x * P.block > 0xffffffffu) return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu n=%zu exceed the grid", what, t, n);
    return 0;
}

extern "C" int w4a16_plan_w8a8(size_t n, size_t k, size_t t, int cu_count, int glu, char* kernel, size_t cap, size_t* workgroups, int* waves, int* k_slices) {
    if (cu_count <= 0 || (kernel && cap < sizeof(W8Launch::kernel)))
        return w4_fail(W4A16_ERR_ARG, "plan_w8a8: cus=%d, %zu bytes for a name of up to %zu", cu_count, cap, sizeof(W8Launch::kernel));
    W4_TRY(w4_q8_check_rows("plan_w8a8", t, k));
    if (n == 0 || n > 0x7fffff00u || (glu && n % 32 != 0))
        return w4_fail(W4A16_ERR_SHAPE, "plan_w8a8: n=%zu outside 1..2^31-256, or gated and no multiple of 32", n);
    W8Launch P;
    W4_TRY(plan_w8a8("plan_w8a8", n, k, t, (size_t)cu_count, glu != 0, &P));
    if (kernel) memcpy(kernel, P.kernel, sizeof P.kernel);
    if (workgroups) *workgroups = P.grid_x * P.grid_y;
    if (waves) *waves = P.block / 64;
    if (k_slices) *k_slices = P.nks;
    return 0;
}

static int launch_w8a8(w4a16_ctx* ctx, const W8Lin& L, const W8Launch& P, uint64_t q, uint64_t s, size_t t, uint64_t y, int y_type, int act) {
    if (P.nks > 1) W4_TRY(w4_split_workspace(ctx, P.part_bytes, P.tickets));
    uint64_t wt = L.q, ws = L.s, part = ctx->w8_part, tickets = ctx->w8_tickets;
    int ni = (int)L.n, kti = (int)k_tiles(L.k), ti = (int)t, r = (int)w4_q8_tile_rows(t), wi = P.block / 64, ksi = P.nks, band = P.band;
    void* few[] = {&wt, &ws, &q, &s, &y, &ni, &kti, &ti, &r, &y_type, &act, &wi, &ksi, &part, &tickets};
    void* tiles[] = {&wt, &ws, &q, &s, &y, &ni, &kti, &ti, &y_type, &act, &ksi, &band, &part, &tickets};
    return w4_launch(ctx, P.kernel, (unsigned)P.grid_x, (unsigned)P.grid_y, (unsigned)P.block, 0, P.band ? tiles : few);
}

static int forward_w8a8(w4a16_ctx* ctx, const char* api, const char* name, uint64_t x, int x_type, size_t ldx, uint64_t xs, size_t t, uint64_t y,
                        int y_type, int act) {
    const W8Lin* L = nullptr;
    W4_TRY(find_w8(ctx, name, &L));
    if (!x || !y) return w4_fail(W4A16_ERR_ARG, "%s %s: null operand", api, name);
    if (x_type != W4A16_Q8 && !w4_float_type(x_type))
        return w4_fail(W4A16_ERR_ARG, "%s %s: x type %d (0 = f32, 1 = f16, 2 = bf16, 3 = quantised rows)", api, name, x_type);
    if (!w4_float_type(y_type)) return w4_fail(W4A16_ERR_ARG, "%s %s: y type %d (0 = f32, 1 = f16, 2 = bf16)", api, name, y_type);
    W4_TRY(w4_q8_check_rows(api, t, L->k));
    if (x_type == W4A16_Q8 ? !xs || ldx != 0 : xs != 0)
        return w4_fail(W4A16_ERR_ARG, "%s %s: quantised rows come with their scales and without a row stride, others without scales", api, name);
    if (act >= 0 && L->n % 32 != 0)
        return w4_fail(W4A16_ERR_SHAPE, "%s %s: n=%zu must be a multiple of 32 (gate and values of whole row blocks)", api, name, L->n);
    if (x_type != W4A16_Q8) {
        if (ldx == 0) ldx = L->k;
        if (ldx < L->k) return w4_fail(W4A16_ERR_SHAPE, "%s %s: ldx=%zu below k=%zu", api, name, ldx, L->k);
    }
    if (y % w4_type_bytes(y_type) || x % (x_type == W4A16_Q8 ? 16 : w4_type_bytes(x_type)) || xs % 4)
        return w4_fail(W4A16_ERR_ARG, "%s %s: operands must be aligned to their elements, quantised rows to 16 bytes", api, name);
    W8Launch P;
    W4_TRY(plan_w8a8(api, L->n, L->k, t, (size_t)std::max(ctx->cu_count, 1), act >= 0, &P));
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    if (x_type != W4A16_Q8) {
        W4_TRY(w4_ensure(ctx, &ctx->q8, &ctx->q8_cap, w4a16_q8_bytes(t, L->k)));
        W4_TRY(w4_ensure(ctx, &ctx->q8_scales, &ctx->q8_scales_cap, std::max<size_t>(t * 4, 256)));
        W4_TRY(quant_rows(ctx, x, x_type, ldx, t, L->k, ctx->q8, ctx->q8_scales));
        x = ctx->q8;
        xs = ctx->q8_scales;
    }
    return launch_w8a8(ctx, *L, P, x, xs, t, y, y_type, act);
}

extern "C" int w4a16_lin_forward_w8a8(w4a16_ctx* ctx, const char* name, uint64_t x_dev, int x_type, size_t ldx, uint64_t xs_dev, size_t t,
                                      uint64_t y_dev, int y_type) {
    return forward_w8a8(ctx, "lin_forward_w8a8", name, x_dev, x_type, ldx, xs_dev, t, y_dev, y_type, -1);
}

extern "C" int w4a16_lin_forward_w8a8_glu(w4a16_ctx* ctx, const char* name, uint64_t x_dev, int x_type, size_t ldx, uint64_t xs_dev, size_t t,
                                          uint64_t y_dev, int y_type, int act) {
    if (act != W4A16_ACT_SILU && act != W4A16_ACT_GELU_TANH)
        return w4_fail(W4A16_ERR_ARG, "lin_forward_w8a8_glu %s: activation %d (0 = silu, 1 = gelu, tanh form)", name ? name : "", act);
    return forward_w8a8(ctx, "lin_forward_w8a8_glu", name, x_dev, x_type, ldx, xs_dev, t, y_dev, y_type, act);
}
