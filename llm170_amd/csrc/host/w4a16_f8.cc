// FP8 linears with a scale for each block of 128: registration, quantisation of activation rows, regime dispatch (kernels/f8_quant.hip, kernels/f8.hip).
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <memory>
#include <new>

#include "w4a16_internal.h"

static inline unsigned ceil_div(size_t a, size_t b) { return (unsigned)((a + b - 1) / b); }

static int quant_rows(w4a16_ctx* ctx, uint64_t x, int x_type, size_t ldx, size_t t, size_t k, uint64_t q, uint64_t s) {
    char sym[64];
    snprintf(sym, sizeof sym, "w4a16_quant_rows_f8_%s", w4_type_name(x_type));
    int ki = (int)k, kb = (int)w4_q8_blocks(k), r = (int)w4_q8_tile_rows(t);
    size_t s_ld = t;
    // a workgroup takes 32, 8 or 2 blocks of 1, 4 or 16 rows
    const size_t most = w4_rows_per_launch(256) * 16;
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        uint64_t x_at = x + at * ldx * w4_type_bytes(x_type), q_at = q + at * kb * 128, s_at = s + at * 4;
        int ti = (int)rows;
        void* params[] = {&x_at, &ldx, &ki, &kb, &r, &q_at, &s_at, &ti, &s_ld};
        W4_TRY(w4_launch(ctx, sym, ceil_div(rows, r), ceil_div(kb, r == 1 ? 32 : r == 4 ? 8 : 2), 256, 0, params));
    }
    return 0;
}

extern "C" int w4a16_quant_rows_f8(w4a16_ctx* ctx, uint64_t x_dev, int x_type, size_t ldx, size_t t, size_t k, uint64_t q_dev, uint64_t s_dev) {
    if (!ctx || !x_dev || !q_dev || !s_dev) return w4_fail(W4A16_ERR_ARG, "quant_rows_f8: null operand");
    if (!w4_float_type(x_type)) return w4_fail(W4A16_ERR_ARG, "quant_rows_f8: x type %d (0 = f32, 1 = f16, 2 = bf16)", x_type);
    W4_TRY(w4_q8_check_rows("quant_rows_f8", t, k));
    if (ldx == 0) ldx = k;
    if (ldx < k) return w4_fail(W4A16_ERR_SHAPE, "quant_rows_f8: ldx=%zu below k=%zu", ldx, k);
    if (x_dev % w4_type_bytes(x_type) || s_dev % 4 || q_dev % 16)
        return w4_fail(W4A16_ERR_ARG, "quant_rows_f8: x and s must be aligned to their elements, q to 16 bytes");
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    return quant_rows(ctx, x_dev, x_type, ldx, t, k, q_dev, s_dev);
}

extern "C" int w4a16_norm_resid_f8(w4a16_ctx* ctx, uint64_t x_dev, uint64_t nw_dev, uint64_t ab_dev, uint64_t q_dev, uint64_t s_dev, size_t t,
                                   size_t w_off, size_t hidden) {
    if (!ctx || !x_dev || !nw_dev || !ab_dev || !q_dev || !s_dev) return w4_fail(W4A16_ERR_ARG, "norm_resid_f8: null operand");
    if (hidden == 0 || hidden > 8192) return w4_fail(W4A16_ERR_SHAPE, "norm_resid_f8: hidden=%zu outside 1..8192", hidden);
    if (w_off > 0x7fffffffu - hidden) return w4_fail(W4A16_ERR_SHAPE, "norm_resid_f8: w_off=%zu too large", w_off);
    W4_TRY(w4_q8_check_rows("norm_resid_f8", t, hidden));
    if (x_dev % 4 || nw_dev % 4 || ab_dev % 4 || s_dev % 4 || q_dev % 16)
        return w4_fail(W4A16_ERR_ARG, "norm_resid_f8: f32 operands must be aligned to 4 bytes, q to 16");
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    int wo = (int)w_off, h = (int)hidden, kb = (int)w4_q8_blocks(hidden), r = (int)w4_q8_tile_rows(t);
    size_t s_ld = t;
    const size_t most = w4_rows_per_launch(256);
    for (size_t at = 0; at < t; at += most) {
        const size_t rows = std::min(most, t - at);
        uint64_t x_at = x_dev + at * hidden * 4, ab_at = ab_dev + at * hidden * 4, q_at = q_dev + at * kb * 128, s_at = s_dev + at * 4;
        int ti = (int)rows;
        void* params[] = {&x_at, &nw_dev, &ab_at, &q_at, &s_at, &wo, &h, &kb, &r, &ti, &s_ld};
        W4_TRY(w4_launch(ctx, "w4a16_norm_resid_f8", r == 16 ? ceil_div(rows, 128) * 128 : (unsigned)rows, 1, 256, 0, params));
    }
    return 0;
}

// ------------------------------------------------------------------------------------------------ registration
static void free_f8(w4a16_ctx* ctx, F8Lin& L) {
    (void)w4a16_free(ctx, L.q);
    (void)w4a16_free(ctx, L.s);
    L = F8Lin();
}

extern "C" int w4a16_upload_lin_f8(w4a16_ctx* ctx, const char* name, const void* q, size_t qlen_bytes, const void* s, size_t slen_bytes, size_t n,
                                   size_t k, int s_type) {
    if (!ctx || !name || !q || !s) return w4_fail(W4A16_ERR_ARG, "upload_lin_f8: null argument");
    if (!w4_float_type(s_type)) return w4_fail(W4A16_ERR_ARG, "upload_lin_f8 %s: scale type %d (0 = f32, 1 = f16, 2 = bf16)", name, s_type);
    const bool fits = n != 0 && n <= 0x7fffff00u && k != 0 && k <= kW4Q8MaxK;
    const size_t kb = fits ? w4_q8_blocks(k) : 0, count = fits ? (n + 127) / 128 * kb : 0;
    if (!fits || qlen_bytes != n * k || slen_bytes != count * w4_type_bytes(s_type))
        return w4_fail(W4A16_ERR_SHAPE, "upload_lin_f8 %s: q=%zu s=%zu bytes for n=%zu k=%zu (k up to %d, a scale for each 128 x 128)", name, qlen_bytes,
                       slen_bytes, n, k, kW4Q8MaxK);
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    F8Lin L;
    L.n = n;
    L.k = k;
    const size_t chunks = (n + 15) / 16 * kb * 128;
    std::unique_ptr<float[]> scales(new (std::nothrow) float[count]());
    if (!scales) return w4_fail(W4A16_ERR_ARG, "upload_lin_f8 %s: no host memory for %zu scales", name, count);
    for (size_t i = 0; i < count; i++) scales[i] = w4_scale_at(s, s_type, i);
    uint64_t raw = 0;
    int rc = w4a16_alloc(ctx, chunks * 16, &L.q);
    if (!rc) rc = w4a16_alloc(ctx, count * 4, &L.s);
    if (!rc) rc = w4a16_alloc(ctx, qlen_bytes, &raw);
    if (!rc) rc = w4a16_h2d(ctx, raw, q, qlen_bytes);
    if (!rc) rc = w4a16_h2d(ctx, L.s, scales.get(), count * 4);
    if (!rc) {
        size_t ns = n, cs = chunks;
        int ki = (int)k, kti = (int)kb * 2;
        void* params[] = {&raw, &L.q, &ns, &ki, &kti, &cs};
        rc = w4_launch(ctx, "w4a16_tile_w8", (unsigned)std::min<size_t>((chunks + 255) / 256, 65536), 1, 256, 0, params);  // bytes, whatever they stand for
    }
    if (!rc) rc = w4a16_sync(ctx);
    const std::string keep = rc ? w4_err_save() : std::string();
    (void)w4a16_free(ctx, raw);
    if (rc) {
        free_f8(ctx, L);
        w4_err_restore(keep);
        return rc;
    }
    auto it = ctx->f8lins.find(std::string_view(name));
    if (it != ctx->f8lins.end()) {
        free_f8(ctx, it->second);
        ctx->scratch_gen++;  // graphs captured so far hold the old weights' address
        it->second = L;
    } else {
        ctx->f8lins.emplace(name, L);
    }
    return 0;
}

static int find_f8(w4a16_ctx* ctx, const char* name, const F8Lin** out) {
    if (!ctx || !name) return w4_fail(W4A16_ERR_ARG, "lin_f8: null argument");
    auto it = ctx->f8lins.find(std::string_view(name));
    if (it == ctx->f8lins.end()) return w4_fail(W4A16_ERR_NOT_FOUND, "lin_f8 %s: not registered", name);
    *out = &it->second;
    return 0;
}

extern "C" int w4a16_lin_f8_info(w4a16_ctx* ctx, const char* name, size_t* n, size_t* k) {
    const F8Lin* L = nullptr;
    W4_TRY(find_f8(ctx, name, &L));
    if (n) *n = L->n;
    if (k) *k = L->k;
    return 0;
}

// ------------------------------------------------------------------------------------------------ forward
// Launch of the kernel for groups of up to 64 rows: row blocks per workgroup, waves, k slices; a function of the shape alone.
// Prices in us, fitted to 226 shapes (512 x 1024 to 65536 x 1024, 1000 x 17408, 1 to 1000 rows): with those of the tiles they pick launches 1 % above the best on average.
struct F8Skinny {
    int rb = 1, waves = 8, nks = 1;
    double price = 0.0;
};

static F8Skinny plan_skinny(size_t n, size_t k, size_t t, size_t cus, bool glu) {
    const size_t kt = w4_q8_blocks(k) * 2, blocks16 = (n + 15) / 16;
    const size_t groups = (t + 63) / 64;
    const int tt = (int)((t + 16 * groups - 1) / (16 * groups));
    F8Skinny best;
    best.price = 1e30;
    // Four row blocks a workgroup pay with 17 to 48 rows alone (5120 x 17408 at 40 24.3 us, two 27.9; at 16 none do; at 64 their sums leave no room for loads in flight)
    for (int rb = tt == 2 || tt == 3 ? 4 : 2; rb >= (glu ? 2 : 1); rb /= 2) {
        for (int nks = 1; nks <= 8; nks++) {
            const size_t grid = (blocks16 + rb - 1) / rb * nks * groups;
            if (nks > 1 && ((size_t)nks * 8 > kt || grid > 4 * cus)) break;
            const double run = (double)kt / nks, load = (double)grid / (double)cus, rounds = 0.92 * std::max(1.0, 0.89 * std::ceil(load) + 0.11 * load) + 0.08;
            const double products = rounds * run * (rb + 0.62 * (t <= 4 ? 0.25 : tt)) * 0.024;
            const double tiles = (double)blocks16 * (double)kt, loads = tiles * 0.000146 * (1.0 + 0.104 * tt * groups / rb);
            const double join = nks == 1 ? 0.0 : 2.5 + 0.24e-6 * nks * n * t * 8;
            F8Skinny p;
            p.rb = rb;
            p.nks = nks;
            p.waves = (grid > cus && t > 16) || run <= 16 ? 4 : 8;  // 34816 x 5120 gated at 40 rows: 4 waves 48.3 us, 8 64.1
            p.waves = (int)std::min<size_t>(p.waves, std::max<size_t>(kt / 2, 1));
            p.price = 2.7 + std::max(products, loads) + join + 0.22 * rb * tt + 0.000032 * tiles * tt * groups / rb;
            if (p.price < best.price) best = p;
        }
    }
    return best;
}

// Launch of a tiled kernel: rows and columns (of weights) per tile, k slices; a function of the shape alone.  Prices as above.
struct F8Tiled {
    int bm = 64, bn = 128, nks = 1;
    double price = 0.0;
};

static F8Tiled plan_tiled(size_t n, size_t k, size_t t, size_t cus, bool exact) {
    // of 64 k: one workgroup of a CU, all of them
    struct Tile { int bm, bn, per_cu; double alone, full; };
    static const Tile kExact[] = {{64, 128, 3, 0.325, 0.588}, {64, 256, 2, 0.479, 0.610}}, kE4m3[] = {{64, 128, 4, 0.213, 0.549}, {128, 256, 2, 0.437, 0.857}};
    const double start = exact ? 5.7 : 6.7, whole = exact ? 0.82 : 0.77, per_slice = exact ? 1.3 : 1.23, per_load = exact ? 13.7 : 9.7;
    const size_t kt = w4_q8_blocks(k) * 2;
    F8Tiled best;
    best.price = 1e30;
    for (int i = 0; i < 2; i++) {
        const Tile& T = exact ? kExact[i] : kE4m3[i];
        for (int nks = 1; nks <= 8; nks++) {
            const size_t grid = (t + T.bm - 1) / T.bm * ((n + T.bn - 1) / T.bn) * nks;
            if (nks > 1 && ((size_t)nks * 8 > kt || grid > T.per_cu * cus)) break;
            const double load = (double)grid / (double)cus, rounds = load / T.per_cu;
            const double per_k = rounds <= 1.0 ? T.alone + (T.full - T.alone) * (std::ceil(load) - 1.0) / (T.per_cu - 1)
                                               : T.full * (whole * std::ceil(rounds) + (1.0 - whole) * rounds);
            F8Tiled p;
            p.bm = T.bm;
            p.bn = T.bn;
            p.nks = nks;
            p.price = start + (double)((kt + nks - 1) / nks) * per_k + (nks > 1 ? (per_slice * nks + per_load * load) * T.bm * T.bn / 32768.0 : 0.0);
            if (p.price < best.price) best = p;
        }
    }
    return best;
}

// The kernel that t rows through a linear go to, its grid, and the scratch of its k slices
struct F8Launch {
    char kernel[64] = "";
    size_t grid_x = 0, grid_y = 1, tickets = 0, part_bytes = 0;
    int block = 256, nks = 1, band = 0;  // band: tile rows of a band, 0 = the kernel for groups of up to 64 rows
    size_t lds_x = 0;                    // bytes of LDS for rows of floats that the kernel quantises (132 a block: the numbers and a scale); 0: it takes quantised rows
};

static int plan_f8(const char* what, size_t n, size_t k, size_t t, size_t cus, bool glu, int x_type, int y_type, F8Launch* out) {
    F8Launch& P = *out;
    const bool exact = y_type == W4A16_F32 || t <= 64 || (glu && t <= 1024);  // the products' own precision: kernels/f8.hip
    const F8Skinny few = plan_skinny(n, k, t, cus, glu);
    const F8Tiled tiles = plan_tiled(n, k, t, cus, exact);
    if (t <= 16 || (t <= 1024 && few.price < tiles.price)) {
        const size_t groups = (t + 63) / 64;  // of as many rows each as can be
        const int tt = (int)((t + 16 * groups - 1) / (16 * groups));
        const size_t blocks16 = (n + 15) / 16;
        // Floats are quantised by the kernel itself, each workgroup its k slice of them, where that takes less than a launch before it does (1.7 to 2.5 us): a few blocks of
        // 128, once or, with one or two rows, a few times a CU.  4096 x 4096 at 1 row 7.1 us, 6.0 and 2.1 with a launch of its own; 65536 x 1024 at 8 rows 17.2, 13.8 and 2.3.
        const size_t blocks = (w4_q8_blocks(k) + few.nks - 1) / few.nks * t, grid = (glu ? (blocks16 / 2 + few.rb / 2 - 1) / (few.rb / 2) : (blocks16 + few.rb - 1) / few.rb) * few.nks;
        if (x_type != W4A16_F8 && t <= 16 && blocks <= kW4F8FloatBlocks && grid <= (t <= 2 ? 4 * cus : cus)) P.lds_x = blocks * 132;
        char rows[8];
        snprintf(rows, sizeof rows, "t%d", tt);
        snprintf(P.kernel, sizeof P.kernel, "w4a16_f8_skinny_r%d_%s%s", few.rb, P.lds_x ? w4_type_name(x_type) : rows, glu ? "_glu" : "");
        P.nks = few.nks;
        P.grid_x = glu ? (blocks16 / 2 + few.rb / 2 - 1) / (few.rb / 2) : (blocks16 + few.rb - 1) / few.rb;
        P.grid_y = few.nks * groups;
        P.block = few.waves * 64;
        P.tickets = P.grid_x * groups;
        P.part_bytes = P.tickets * few.nks * few.rb * tt * 1024;
    } else {
        if (exact) snprintf(P.kernel, sizeof P.kernel, "w4a16_f8_exact_n%d%s", tiles.bn, glu ? "_glu" : "");
        else snprintf(P.kernel, sizeof P.kernel, "w4a16_f8_tiled_m%d%s", tiles.bm, glu ? "_glu" : "");
        P.nks = tiles.nks;
        P.tickets = (t + tiles.bm - 1) / tiles.bm * ((n + tiles.bn - 1) / tiles.bn);
        P.part_bytes = P.tickets * tiles.nks * tiles.bm * tiles.bn * 4;
        P.grid_x = (P.tickets * tiles.nks + 7) / 8 * 8;
        P.band = 1024 / tiles.bm;  // 1024 rows of tiles share their weights in the L2
    }
    if (P.grid_x * P.block > 0xffffffffu) return w4_fail(W4A16_ERR_SHAPE, "%s: t=%zu n=%zu exceed the grid", what, t, n);
    return 0;
}

extern "C" int w4a16_plan_f8(size_t n, size_t k, size_t t, int cu_count, int glu, int x_type, int y_type, char* kernel, size_t cap, size_t* workgroups,
                             int* waves, int* k_slices) {
    if (cu_count <= 0 || (kernel && cap < sizeof(F8Launch::kernel)))
        return w4_fail(W4A16_ERR_ARG, "plan_f8: cus=%d, %zu bytes for a name of up to %zu", cu_count, cap, sizeof(F8Launch::kernel));
    if (x_type != W4A16_F8 && !w4_float_type(x_type)) return w4_fail(W4A16_ERR_ARG, "plan_f8: x type %d (0 = f32, 1 = f16, 2 = bf16, 4 = rows quantised to e4m3)", x_type);
    if (!w4_float_type(y_type)) return w4_fail(W4A16_ERR_ARG, "plan_f8: y type %d (0 = f32, 1 = f16, 2 = bf16)", y_type);
    W4_TRY(w4_q8_check_rows("plan_f8", t, k));
    if (n == 0 || n > 0x7fffff00u || (glu && n % 256 != 0))
        return w4_fail(W4A16_ERR_SHAPE, "plan_f8: n=%zu outside 1..2^31-256, or gated and no multiple of 256", n);
    F8Launch P;
    W4_TRY(plan_f8("plan_f8", n, k, t, (size_t)cu_count, glu != 0, x_type, y_type, &P));
    if (kernel) memcpy(kernel, P.kernel, sizeof P.kernel);
    if (workgroups) *workgroups = P.grid_x * P.grid_y;
    if (waves) *waves = P.block / 64;
    if (k_slices) *k_slices = P.nks;
    return 0;
}

static int launch_f8(w4a16_ctx* ctx, const F8Lin& L, const F8Launch& P, uint64_t q, uint64_t s, size_t ldx, size_t t, uint64_t y, int y_type, int act) {
    if (P.nks > 1) W4_TRY(w4_split_workspace(ctx, P.part_bytes, P.tickets));
    uint64_t wt = L.q, ws = L.s, part = ctx->w8_part, tickets = ctx->w8_tickets;
    int ni = (int)L.n, ki = (int)L.k, kb = (int)w4_q8_blocks(L.k), ti = (int)t, r = (int)w4_q8_tile_rows(t), wi = P.block / 64, ksi = P.nks, band = P.band;
    void* few[] = {&wt, &ws, &q, &s, &y, &ni, &kb, &ti, &r, &y_type, &act, &wi, &ksi, &part, &tickets};
    void* floats[] = {&wt, &ws, &q, &ldx, &ki, &y, &ni, &kb, &ti, &y_type, &act, &wi, &ksi, &part, &tickets};
    void* tiles[] = {&wt, &ws, &q, &s, &y, &ni, &kb, &ti, &y_type, &act, &ksi, &band, &part, &tickets};
    return w4_launch(ctx, P.kernel, (unsigned)P.grid_x, (unsigned)P.grid_y, (unsigned)P.block, (unsigned)P.lds_x, P.band ? tiles : P.lds_x ? floats : few);
}

static int forward_f8(w4a16_ctx* ctx, const char* api, const char* name, uint64_t x, int x_type, size_t ldx, uint64_t xs, size_t t, uint64_t y,
                      int y_type, int act) {
    const F8Lin* L = nullptr;
    W4_TRY(find_f8(ctx, name, &L));
    if (!x || !y) return w4_fail(W4A16_ERR_ARG, "%s %s: null operand", api, name);
    if (x_type != W4A16_F8 && !w4_float_type(x_type))
        return w4_fail(W4A16_ERR_ARG, "%s %s: x type %d (0 = f32, 1 = f16, 2 = bf16, 4 = rows quantised to e4m3)", api, name, x_type);
    if (!w4_float_type(y_type)) return w4_fail(W4A16_ERR_ARG, "%s %s: y type %d (0 = f32, 1 = f16, 2 = bf16)", api, name, y_type);
    W4_TRY(w4_q8_check_rows(api, t, L->k));
    if (x_type == W4A16_F8 ? !xs || ldx != 0 : xs != 0)
        return w4_fail(W4A16_ERR_ARG, "%s %s: quantised rows come with their scales and without a row stride, others without scales", api, name);
    if (act >= 0 && L->n % 256 != 0)
        return w4_fail(W4A16_ERR_SHAPE, "%s %s: n=%zu must be a multiple of 256 (gate and values of whole blocks of 128)", api, name, L->n);
    if (x_type != W4A16_F8) {
        if (ldx == 0) ldx = L->k;
        if (ldx < L->k) return w4_fail(W4A16_ERR_SHAPE, "%s %s: ldx=%zu below k=%zu", api, name, ldx, L->k);
    }
    if (y % w4_type_bytes(y_type) || x % (x_type == W4A16_F8 ? 16 : w4_type_bytes(x_type)) || xs % 4)
        return w4_fail(W4A16_ERR_ARG, "%s %s: operands must be aligned to their elements, quantised rows to 16 bytes", api, name);
    F8Launch P;
    W4_TRY(plan_f8(api, L->n, L->k, t, (size_t)std::max(ctx->cu_count, 1), act >= 0, x_type, y_type, &P));
    W4_TRY(w4_hip(hipSetDevice(ctx->device), "hipSetDevice"));
    if (x_type != W4A16_F8 && !P.lds_x) {
        W4_TRY(w4_ensure(ctx, &ctx->q8, &ctx->q8_cap, w4a16_q8_bytes(t, L->k)));
        W4_TRY(w4_ensure(ctx, &ctx->q8_scales, &ctx->q8_scales_cap, std::max<size_t>(t * w4_q8_blocks(L->k) * 4, 256)));
        W4_TRY(quant_rows(ctx, x, x_type, ldx, t, L->k, ctx->q8, ctx->q8_scales));
        x = ctx->q8;
        xs = ctx->q8_scales;
    }
    return launch_f8(ctx, *L, P, x, xs, ldx, t, y, y_type, act);
}

extern "C" int w4a16_lin_forward_f8(w4a16_ctx* ctx, const char* name, uint64_t x_dev, int x_type, size_t ldx, uint64_t xs_dev, size_t t, uint64_t y_dev,
                                    int y_type) {
    return forward_f8(ctx, "lin_forward_f8", name, x_dev, x_type, ldx, xs_dev, t, y_dev, y_type, -1);
}

extern "C" int w4a16_lin_forward_f8_glu(w4a16_ctx* ctx, const char* name, uint64_t x_dev, int x_type, size_t ldx, uint64_t xs_dev, size_t t,
                                        uint64_t y_dev, int y_type, int act) {
    if (act != W4A16_ACT_SILU && act != W4A16_ACT_GELU_TANH)
        return w4_fail(W4A16_ERR_ARG, "lin_forward_f8_glu %s: activation %d (0 = silu, 1 = gelu, tanh form)", name ? name : "", act);
    return forward_f8(ctx, "lin_forward_f8_glu", name, x_dev, x_type, ldx, xs_dev, t, y_dev, y_type, act);
}
