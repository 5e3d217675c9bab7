// libartread.so — operators that read the passages a search found (include/artread.h).  gfx950 only.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../../include/artread.h"
#include "artread_attend.h"
#include "artread_attend_grad.h"
#include "artread_embed.h"

static thread_local char g_read_err[512] = "";

static int read_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_read_err, sizeof(g_read_err), fmt, ap);
    va_end(ap);
    return code;
}

#define READ_HIP(expr)                                                                          \
    do {                                                                                        \
        hipError_t e__ = (expr);                                                                \
        if (e__ != hipSuccess)                                                                  \
            return read_fail(ARTREAD_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e__), \
                             __FILE__, __LINE__);                                               \
    } while (0)
#define READ_ARG(cond, ...)                                          \
    do {                                                             \
        if (!(cond)) return read_fail(ARTREAD_ERR_ARG, __VA_ARGS__); \
    } while (0)

struct ReadDeviceGuard {
    int prev = -1, dev;
    hipError_t err = hipSuccess;
    explicit ReadDeviceGuard(int d) : dev(d) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != dev) err = hipSetDevice(dev);
        if (err != hipSuccess) (void)hipGetLastError();   // reported here, not by the next call
    }
    ~ReadDeviceGuard() {
        if (prev >= 0 && prev != dev) (void)hipSetDevice(prev);
    }
};

extern "C" const char* artread_last_error(void) { return g_read_err; }

static constexpr int64_t kLimit = (int64_t)1 << 31;
static constexpr int64_t kStrideLimit = (int64_t)1 << 40;
static constexpr int64_t kRowLimit = (int64_t)1 << 24;   // the rows of a tile stay within 32 bits of bytes
static bool tile_fits(int64_t row, int64_t head, int64_t share) { return row < kRowLimit && head * share < 32 * kRowLimit; }
static int elem_bytes(int dtype) { return dtype == ARTREAD_F32 ? 4 : 2; }
static bool aligned(const void* p, uint64_t to) { return ((uintptr_t)p) % to == 0; }
static int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// ---- embedding ------------------------------------------------------------------------------------
static int check_tokens(const void* tokens, int token_bytes, const int32_t* lengths, int64_t n, int64_t len,
                        int64_t vocab, int64_t dim, int64_t vocab_base, Tokens* T) {
    READ_ARG(tokens, "tokens is NULL");
    READ_ARG(token_bytes == 4 || token_bytes == 8, "token_bytes must be 4 or 8 (got %d)", token_bytes);
    READ_ARG(aligned(tokens, token_bytes) && aligned(lengths, 4), "misaligned tokens or lengths");
    READ_ARG(n >= 1 && len >= 1 && n < kLimit && len < kLimit && n * len < kLimit,
             "n %lld x len %lld must be in [1, 2^31)", (long long)n, (long long)len);
    READ_ARG(vocab >= 1 && vocab < kLimit, "vocab %lld must be in [1, 2^31)", (long long)vocab);
    READ_ARG(dim >= 1 && dim <= (1 << 20), "dim %lld must be in [1, 2^20]", (long long)dim);
    T->tokens = tokens;
    T->lengths = lengths;
    T->len = (uint32_t)len;
    T->inv_len = len == 1 ? 0xffffffffu : (uint32_t)(((uint64_t)1 << 32) / (uint64_t)len);
    T->vocab = vocab;
    T->vocab_base = vocab_base;
    T->positions = n * len;
    return 0;
}

template <typename TT, typename OT, typename IDX, int EPV>
static void launch_embed(const void* table, int64_t stride, const Tokens& T, float scale, void* out, int dim,
                         hipStream_t st) {
    const int cpr = dim / EPV, rpp = cpr < 256 ? 256 / cpr : 1;
    const int threads = cpr < 256 ? (int)round_up((int64_t)cpr * rpp, 64) : 256;
    const int64_t want = (T.positions + (int64_t)rpp * kEmbedRows - 1) / ((int64_t)rpp * kEmbedRows);
    const unsigned grid = (unsigned)(want < (1 << 22) ? want : (1 << 22));
    hipLaunchKernelGGL((embed_kernel<TT, OT, IDX, EPV>), dim3(grid), dim3(threads), 0, st, (const TT*)table, stride, T,
                       scale, (OT*)out, dim, cpr, rpp);
}

template <typename TT, typename OT>
static void embed_any(const void* table, int64_t stride, const Tokens& T, int token_bytes, float scale, void* out,
                      int dim, hipStream_t st) {
    // chunks of 16 bytes of output where rows allow them, else pairs of elements, else one
    constexpr int W = 16 / sizeof(OT);
    const bool wide = dim % W == 0 && stride % (16 / (int)sizeof(TT)) == 0 && aligned(table, 16) && aligned(out, 16);
    const bool pairs = dim % 2 == 0 && stride % 2 == 0 && aligned(table, 2 * sizeof(TT)) && aligned(out, 2 * sizeof(OT));
#define EMBED(IDX)                                                                              \
    do {                                                                                        \
        if (wide) launch_embed<TT, OT, IDX, W>(table, stride, T, scale, out, dim, st);          \
        else if (pairs) launch_embed<TT, OT, IDX, 2>(table, stride, T, scale, out, dim, st);    \
        else launch_embed<TT, OT, IDX, 1>(table, stride, T, scale, out, dim, st);               \
    } while (0)
    if (token_bytes == 4) EMBED(int32_t);
    else EMBED(int64_t);
#undef EMBED
}

extern "C" int artread_embed(int device, const void* table, int table_dtype, int64_t vocab, int64_t dim,
                             int64_t table_stride, const void* tokens, int token_bytes, const int32_t* lengths,
                             int64_t n, int64_t len, int64_t vocab_base, float scale, void* out, int out_dtype,
                             void* stream) {
    Tokens T;
    const int rc = check_tokens(tokens, token_bytes, lengths, n, len, vocab, dim, vocab_base, &T);
    if (rc) return rc;
    READ_ARG(table && out, "table or out is NULL");
    READ_ARG(table_stride >= dim || vocab == 1, "table_stride %lld is below dim %lld", (long long)table_stride,
             (long long)dim);
    READ_ARG(table_dtype >= 0 && table_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, "unknown element type");
    READ_ARG(out_dtype == table_dtype || table_dtype == ARTREAD_F32,
             "out must have the table's type, or f16 / bf16 of an f32 table");
    READ_ARG(aligned(table, elem_bytes(table_dtype)) && aligned(out, elem_bytes(out_dtype)), "misaligned pointer");
    READ_ARG(isfinite(scale), "scale must be finite");
    ReadDeviceGuard g(device);
    READ_HIP(g.err);
    hipStream_t st = (hipStream_t)stream;
    if (table_dtype == ARTREAD_F16) embed_any<f16, f16>(table, table_stride, T, token_bytes, scale, out, (int)dim, st);
    else if (table_dtype == ARTREAD_BF16) embed_any<bf16, bf16>(table, table_stride, T, token_bytes, scale, out, (int)dim, st);
    else if (out_dtype == ARTREAD_F16) embed_any<float, f16>(table, table_stride, T, token_bytes, scale, out, (int)dim, st);
    else if (out_dtype == ARTREAD_BF16) embed_any<float, bf16>(table, table_stride, T, token_bytes, scale, out, (int)dim, st);
    else embed_any<float, float>(table, table_stride, T, token_bytes, scale, out, (int)dim, st);
    READ_HIP(hipGetLastError());
    return 0;
}

// Sort digits of at most nine bits; one chunk up to kSortAlone positions, else at most 256 of at least 4,096.
static SortPlan sort_plan(int64_t vocab, int64_t positions) {
    SortPlan P;
    int bits = 1;
    while (bits < 31 && ((int64_t)1 << bits) < vocab) ++bits;
    P.passes = (bits + 8) / 9;
    P.bits = (bits + P.passes - 1) / P.passes;
    P.chunk = round_up(positions <= kSortAlone ? positions : (positions + 255) / 256, kSortThreads);
    if (positions > kSortAlone && P.chunk < 4096) P.chunk = 4096;
    P.blocks = (int)((positions + P.chunk - 1) / P.chunk);
    return P;
}

// Ranges of 128 positions where that many fill the chip, down to 8 where not: the join of a token's partial sums is
// as long as they are many (2,048 x 256 positions of 768 f16: join 12 us with 128, 19 with 64, 33 with 32; sums alike).
static int sum_run(int64_t positions) {
    int run = 128;
    while (run > 8 && positions / run < 4096) run >>= 1;
    return run;
}

struct GradSpace {   // byte offsets into the workspace
    int64_t meta, counts, pairs0, pairs1, chain_end, partial, total;
    int64_t pad_dim;
    int run;
};
static GradSpace grad_space(int64_t vocab, int64_t dim, int64_t positions) {
    const SortPlan P = sort_plan(vocab, positions);
    GradSpace s;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    s.run = sum_run(positions);
    s.pad_dim = round_up(dim, 4);
    s.meta = take(sizeof(SortMeta));
    s.counts = take((int64_t)P.blocks * (1 << P.bits) * 4);
    s.pairs0 = take(positions * 8);
    s.pairs1 = P.passes > 1 ? take(positions * 8) : s.pairs0;
    s.chain_end = take(vocab * 4);
    s.partial = take((positions + s.run - 1) / s.run * 2 * s.pad_dim * 4);
    s.total = at;
    return s;
}

extern "C" int64_t artread_embed_grad_workspace(int64_t vocab, int64_t dim, int64_t n, int64_t len) {
    if (n < 1 || len < 1 || n >= kLimit || len >= kLimit || n * len >= kLimit || vocab < 1 || vocab >= kLimit ||
        dim < 1 || dim > (1 << 20))
        return read_fail(ARTREAD_ERR_ARG, "sizes out of range");
    return grad_space(vocab, dim, n * len).total;
}

template <typename GT, typename OT, int EPV>
static void launch_grad_sums(const void* grad, const Pair* sorted, const SortMeta* meta, const Tokens& T, float scale,
                             void* table, int dim, const GradSpace& s, float* partial, int32_t* chain_end,
                             hipStream_t st) {
    SumPlan S;
    S.run = s.run;
    S.cpr = dim / EPV;
    S.rpp = S.cpr < 256 ? 256 / S.cpr : 1;
    S.pad_dim = s.pad_dim;
    S.workers = (T.positions + s.run - 1) / s.run;
    S.sum_groups = (S.workers + S.rpp - 1) / S.rpp;
    const int threads = S.cpr < 256 ? (int)round_up((int64_t)S.cpr * S.rpp, 64) : 256;
    int64_t clear = (T.vocab + kClearRows - 1) / kClearRows;
    if (clear > (1 << 20)) clear = 1 << 20;
    hipLaunchKernelGGL((grad_sum_kernel<GT, OT, EPV>), dim3((unsigned)(S.sum_groups + clear)), dim3(threads), 0, st,
                       (const GT*)grad, sorted, meta, T.vocab, scale, (OT*)table, dim, S, partial, chain_end);
    if (S.workers > 1)
        hipLaunchKernelGGL((grad_join_kernel<OT>),
                           dim3((unsigned)((S.workers + kJoinWaves - 1) / kJoinWaves), (unsigned)((dim + 255) / 256)),
                           dim3(64 * kJoinWaves), 0, st, sorted, meta, scale, (OT*)table, dim, S, partial, chain_end);
}

template <typename GT, typename OT>
static void grad_sums(const void* grad, const Pair* sorted, const SortMeta* meta, const Tokens& T,
                      float scale, void* table, int dim, const GradSpace& s, float* partial, int32_t* chain_end,
                      hipStream_t st) {
    constexpr int W = 16 / sizeof(GT);
    if (dim % W == 0 && aligned(grad, 16) && aligned(table, 16))
        launch_grad_sums<GT, OT, W>(grad, sorted, meta, T, scale, table, dim, s, partial, chain_end, st);
    else if (dim % 2 == 0 && aligned(grad, 2 * sizeof(GT)) && aligned(table, 2 * sizeof(OT)))
        launch_grad_sums<GT, OT, 2>(grad, sorted, meta, T, scale, table, dim, s, partial, chain_end, st);
    else
        launch_grad_sums<GT, OT, 1>(grad, sorted, meta, T, scale, table, dim, s, partial, chain_end, st);
}

template <typename IDX>
static const Pair* sort_tokens(const Tokens& T, char* ws, const GradSpace& s, hipStream_t st) {
    const SortPlan P = sort_plan(T.vocab, T.positions);
    SortMeta* meta = (SortMeta*)(ws + s.meta);
    uint32_t* counts = (uint32_t*)(ws + s.counts);
    Pair* pairs[2] = {(Pair*)(ws + s.pairs0), (Pair*)(ws + s.pairs1)};
    const dim3 grid((unsigned)P.blocks), block(kSortThreads);
    if (P.blocks == 1) {
        hipLaunchKernelGGL((sort_alone_kernel<IDX>), grid, block, 0, st, T, meta, P, pairs[0], pairs[1]);
        return pairs[(P.passes - 1) & 1];
    }
    for (int pass = 0; pass < P.passes; ++pass) {
        const int shift = pass * P.bits;
        const Pair* in = pairs[(pass + 1) & 1];
        Pair* out = pairs[pass & 1];
        if (pass == 0) {
            hipLaunchKernelGGL((sort_count_kernel<IDX, true>), grid, block, 0, st, T, in, meta, P, shift, counts);
            hipLaunchKernelGGL((sort_place_kernel<IDX, true>), grid, block, 0, st, T, in, meta, P, shift, counts, out);
        } else {
            hipLaunchKernelGGL((sort_count_kernel<IDX, false>), grid, block, 0, st, T, in, meta, P, shift, counts);
            hipLaunchKernelGGL((sort_place_kernel<IDX, false>), grid, block, 0, st, T, in, meta, P, shift, counts, out);
        }
    }
    return pairs[(P.passes - 1) & 1];
}

extern "C" int artread_embed_grad(int device, const void* grad_out, int grad_dtype, const void* tokens, int token_bytes,
                                  const int32_t* lengths, int64_t n, int64_t len, int64_t vocab, int64_t dim,
                                  int64_t vocab_base, float scale, void* grad_table, int table_dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    Tokens T;
    const int rc = check_tokens(tokens, token_bytes, lengths, n, len, vocab, dim, vocab_base, &T);
    if (rc) return rc;
    READ_ARG(grad_out && grad_table && workspace, "grad_out, grad_table or workspace is NULL");
    READ_ARG(grad_dtype >= 0 && grad_dtype <= 2 && table_dtype >= 0 && table_dtype <= 2, "unknown element type");
    READ_ARG(table_dtype == grad_dtype || table_dtype == ARTREAD_F32, "grad_table must have grad_out's type, or f32");
    READ_ARG(aligned(grad_out, elem_bytes(grad_dtype)) && aligned(grad_table, elem_bytes(table_dtype)),
             "misaligned pointer");
    READ_ARG(isfinite(scale), "scale must be finite");
    const GradSpace s = grad_space(vocab, dim, T.positions);
    READ_ARG(aligned(workspace, 16) && workspace_bytes >= s.total, "workspace of %lld bytes, %lld needed, 16-byte aligned",
             (long long)workspace_bytes, (long long)s.total);
    ReadDeviceGuard g(device);
    READ_HIP(g.err);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const Pair* sorted = token_bytes == 4 ? sort_tokens<int32_t>(T, ws, s, st) : sort_tokens<int64_t>(T, ws, s, st);
    READ_HIP(hipGetLastError());
    const SortMeta* meta = (const SortMeta*)(ws + s.meta);
    float* partial = (float*)(ws + s.partial);
    int32_t* ends = (int32_t*)(ws + s.chain_end);
#define SUMS(GT, OT) grad_sums<GT, OT>(grad_out, sorted, meta, T, scale, grad_table, (int)dim, s, partial, ends, st)
    if (grad_dtype == ARTREAD_F32) SUMS(float, float);
    else if (grad_dtype == ARTREAD_F16 && table_dtype == ARTREAD_F16) SUMS(f16, f16);
    else if (grad_dtype == ARTREAD_F16) SUMS(f16, float);
    else if (table_dtype == ARTREAD_BF16) SUMS(bf16, bf16);
    else SUMS(bf16, float);
#undef SUMS
    READ_HIP(hipGetLastError());
    return 0;
}

// ---- attention ------------------------------------------------------------------------------------
static int check_attend(const artread_attend_t* a) {
    READ_ARG(a, "arguments are NULL");
    READ_ARG(a->dtype == ARTREAD_F16 || a->dtype == ARTREAD_BF16, "attention takes f16 or bf16");
    READ_ARG(a->batch >= 1 && a->rows >= 1 && a->passages >= 1 && a->len >= 1 && a->heads >= 1 && a->kv_heads >= 1,
             "batch, rows, passages, len and heads must be positive");
    READ_ARG(a->heads % a->kv_heads == 0, "%lld heads cannot share %lld key heads", (long long)a->heads,
             (long long)a->kv_heads);
    READ_ARG(a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0, "dim %lld must be a multiple of 8 up to 128",
             (long long)a->dim);
    const int64_t sizes[6] = {a->batch, a->rows, a->passages, a->len, a->heads, a->kv_heads};
    for (int i = 0; i < 6; ++i) READ_ARG(sizes[i] < kLimit, "sizes must be below 2^31");
    READ_ARG((double)a->batch * a->rows * a->heads < (double)kLimit &&
                 (double)a->batch * a->passages * a->len * a->kv_heads < (double)kLimit,
             "q and k hold at most 2^31 - 1 rows each");
    READ_ARG(a->passages * a->len <= kLimit - (1 << 20), "a batch entry holds at most 2^31 - 2^20 states");
    READ_ARG(isfinite(a->scale), "scale must be finite");
    const int64_t strides[11] = {a->q_batch, a->q_row, a->q_head, a->k_batch, a->k_passage, a->k_row,
                                 a->k_head, a->v_batch, a->v_passage, a->v_row, a->v_head};
    for (int i = 0; i < 11; ++i)
        READ_ARG(strides[i] >= 0 && strides[i] % 8 == 0 && strides[i] < kStrideLimit,
                 "strides must be multiples of 8 in [0, 2^40)");
    READ_ARG(a->k_row < kRowLimit && a->v_row < kRowLimit && tile_fits(a->q_row, a->q_head, a->heads / a->kv_heads),
             "row strides must be below 2^24, the query heads that share a key head within 2^29 elements");
    return 0;
}
static int check_attend_call(const artread_attend_t* a) {
    const int rc = check_attend(a);
    if (rc) return rc;
    READ_ARG(a->q && a->k && a->v && a->out, "q, k, v or out is NULL");
    READ_ARG(aligned(a->rest, 16), "rest must be 16-byte aligned");
    READ_ARG(aligned(a->lse, 4) && aligned(a->lengths, 4), "misaligned lse or lengths");
    READ_ARG(aligned(a->q, 16) && aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->out, 16),
             "q, k, v and out must be 16-byte aligned");
    return 0;
}
static unsigned grid_of(int64_t items) { return (unsigned)(items < (1 << 22) ? items : (1 << 22)); }

static dim3 grid2(int64_t items) {   // at least `items` workgroups, a multiple of 8 wide: neighbours stay on their XCDs
    const int64_t x = 1 << 16;
    return items <= x ? dim3((unsigned)round_up(items, 8)) : dim3((unsigned)x, (unsigned)((items + x - 1) / x));
}

// How a forward call runs.  Up to 32 rows (64 at 64 columns) of a key head are one wave's, which streams the
// keys; more share their tiles of keys in a workgroup.
struct AttendShape {
    artread_attend_t args;   // as the kernels take them
    bool stream;
    int qb;
    AttendPlan plan;
    Partials partials(void* ws, const artread_attend_t* a) const {
        Partials W;
        W.rows = a->batch * a->kv_heads * plan.row_count;
        W.o = (float*)ws;
        W.ml = (float2*)((char*)ws + round_up(plan.splits * W.rows * a->dim * 4, 256));
        return W;
    }
    int64_t bytes(const artread_attend_t* a) const {
        const int64_t rows = a->batch * a->kv_heads * plan.row_count;
        return plan.splits > 1 ? round_up(plan.splits * rows * a->dim * 4, 256) + round_up(plan.splits * rows * 8, 256) : 0;
    }
};
static void plan_scale(AttendPlan* P, float scale, int dtype) {
    P->c = scale == 0.0f ? 1.0f : fabsf(scale) * kLog2e;
    P->unweight = dtype == ARTREAD_F16 ? exp2f(-Mma<f16>::kWeightLog2) : 1.0f;
    P->q_and = scale == 0.0f ? 0u : 0xffffffffu;
    P->q_xor = scale < 0.0f ? 0x80008000u : 0u;
}
static void plan_share(AttendPlan* P, const artread_attend_t* a) {
    P->share = (uint32_t)(a->heads / a->kv_heads);
    P->inv_share = P->share == 1 ? 0xffffffffu : (uint32_t)(((uint64_t)1 << 32) / P->share);
}
// Passages that lie one behind the other are one long passage where every entry is valid, and one with holes where they
// are short: of a tile of keys a passage of 7 would fill 7 (32 x 100 rows, 100 passages of 7 of 64 columns: forward 39 us
// instead of 164, gradients 81 instead of 620).  Longer ones with lengths keep tiles of their own, which end with them; up
// to 63 packing measured faster where rows are many (1,000 passages of 40, 400 rows: 75 us instead of 107) and is not taken.
// Where passages are packed or one long one, sums run over other tiles than where gaps lie between them: a call's last bits
// depend on its layout there.
constexpr int64_t kPackLength = 32;
static bool few_rows(int64_t row_count, int64_t dim) { return row_count <= (dim <= 64 ? 64 : 32); }
static artread_attend_t pack_passages(const artread_attend_t* given, AttendPlan* P) {
    artread_attend_t a = *given;
    P->pack = P->inv_pack = 0;
    P->pack_passages = a.passages;
    if (a.passages > 1 && (!a.lengths || a.len <= kPackLength) && a.k_passage == a.len * a.k_row && a.v_passage == a.len * a.v_row) {
        if (a.lengths) {
            P->pack = (uint32_t)a.len;
            P->inv_pack = a.len == 1 ? 0xffffffffu : (uint32_t)(((uint64_t)1 << 32) / (uint64_t)a.len);
        }
        a.len *= a.passages;
        a.passages = 1;
    }
    return a;
}
static AttendShape attend_shape(const artread_attend_t* given) {
    AttendShape S;
    AttendPlan& P = S.plan;
    S.args = pack_passages(given, &P);
    const artread_attend_t* a = &S.args;
    plan_share(&P, a);
    P.row_count = a->rows * P.share;
    S.stream = few_rows(P.row_count, a->dim);
    S.qb = S.stream && P.row_count > 32 ? 2 : 1;
    const int block = (S.stream ? 32 : 128) * S.qb, keys = S.stream ? 32 : 64;
    P.row_blocks = (P.row_count + block - 1) / block;
    P.items = a->batch * a->kv_heads * P.row_blocks;
    const int64_t tiles = a->passages * ((a->len + keys - 1) / keys);
    P.walkers = 1;
    if (S.stream) {
        // Workgroups that fill the chip.  By registers two waves share a SIMD, three at 64 columns and 32 rows;
        // a round more evens out the lengths, while each more leaves partial results to join (us, kernel + join,
        // for 8, 12, 16 waves a compute unit: 64 questions x 32 passages x 64 columns 222, 203, 195; 2 x 100 x 128 columns
        // 76, 87, 89; 48 rows 161, 151, 159).
        const int64_t waves = 256 * (a->dim > 64 ? 8 : (S.qb == 2 ? 12 : 16));
        int64_t want = (waves / 4 + P.items - 1) / P.items;
        if (P.items < waves && tiles >= 4) P.walkers = 4;
        else want = 1;
        const int64_t most = tiles / 16;   // parts of at least four tiles a wave: shorter ones cost more in the join than they save
        want = want < most ? want : most;
        P.splits = (int)(want < 1 ? 1 : (want < 256 ? want : 256));
    } else {
        int64_t want = (512 + P.items - 1) / P.items;
        const int64_t most = tiles / 4;
        want = want < most ? want : most;
        P.splits = (int)(want < 1 ? 1 : (want < 256 ? want : 256));
    }
    plan_scale(&P, a->scale, a->dtype);
    return S;
}

extern "C" int64_t artread_attend_workspace(const artread_attend_t* a) {
    const int rc = check_attend(a);
    return rc ? rc : attend_shape(a).bytes(a);
}

template <typename T, int DP>
static void launch_attend(const artread_attend_t* a, const AttendShape& S, const Partials& W, hipStream_t st) {
    const int64_t parts = S.plan.items * S.plan.splits;
    if (S.stream) {
        const dim3 grid = grid2(S.plan.walkers == 1 ? (parts + 3) / 4 : parts);
        if (S.qb == 1) hipLaunchKernelGGL((attend_stream_kernel<T, DP, 1>), grid, dim3(256), 0, st, *a, S.plan, W);
        else if constexpr (DP == 64) hipLaunchKernelGGL((attend_stream_kernel<T, DP, 2>), grid, dim3(256), 0, st, *a, S.plan, W);
    } else {
        const dim3 grid = grid2(parts);
        hipLaunchKernelGGL((attend_tile_kernel<T, DP>), grid, dim3(256), 0, st, *a, S.plan, W);
    }
    if (S.plan.splits > 8)
        hipLaunchKernelGGL((attend_join_kernel<T, 8>), dim3(grid_of(W.rows)), dim3(256), 0, st, *a, S.plan, W);
    else if (S.plan.splits > 1)
        hipLaunchKernelGGL((attend_join_kernel<T, 1>), dim3(grid_of((W.rows + 7) / 8)), dim3(256), 0, st, *a, S.plan, W);
}

extern "C" int artread_attend(int device, const artread_attend_t* a, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    const int rc = check_attend_call(a);
    if (rc) return rc;
    const AttendShape S = attend_shape(a);
    const int64_t need = S.bytes(a);
    READ_ARG(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need),
             "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)need);
    const Partials W = S.partials(workspace, a);
    ReadDeviceGuard g(device);
    READ_HIP(g.err);
    hipStream_t st = (hipStream_t)stream;
    a = &S.args;
    if (a->dtype == ARTREAD_F16) {
        if (a->dim <= 64) launch_attend<f16, 64>(a, S, W, st);
        else launch_attend<f16, 128>(a, S, W, st);
    } else {
        if (a->dim <= 64) launch_attend<bf16, 64>(a, S, W, st);
        else launch_attend<bf16, 128>(a, S, W, st);
    }
    READ_HIP(hipGetLastError());
    return 0;
}

// How a gradient call runs: up to 32 rows of a key head (64 at 64 columns) in one walk over the keys, more in a walk
// over the keys for dQ and one over the rows for dK and dV; each split where its workgroups would not fill the chip.
struct GradShape {
    artread_attend_t args;   // as the kernels take them
    bool fused;
    bool narrow;           // dQ: one wave of 32 rows per workgroup, else four
    AttendPlan q, kv;
    int64_t all_q, all_k;  // elements
    int64_t stats, part;   // byte offsets; the two walks run one after the other and share their parts
    int64_t total;
};
static GradShape grad_shape(const artread_attend_t* given) {
    GradShape S;
    AttendPlan& Q = S.q;
    S.args = pack_passages(given, &Q);
    const artread_attend_t* a = &S.args;
    plan_share(&Q, a);
    Q.row_count = a->rows * Q.share;
    plan_scale(&Q, a->scale, a->dtype);
    Q.pad_rows = round_up(Q.row_count, 64);
    Q.c = a->scale * kLog2e;   // no maximum is taken here: c may be negative or zero
    Q.q_and = 0xffffffffu;
    Q.q_xor = 0u;
    S.kv = Q;
    S.fused = few_rows(Q.row_count, a->dim);
    S.narrow = Q.row_count <= 64;
    const int block = S.narrow ? 32 : 128, keys = S.narrow ? 32 : 64;
    Q.row_blocks = (Q.row_count + block - 1) / block;
    Q.items = a->batch * a->kv_heads * Q.row_blocks;
    int64_t want = ((S.narrow ? 2048 : 512) + Q.items - 1) / Q.items;
    int64_t most = a->passages * ((a->len + keys - 1) / keys) / 4;
    want = want < most ? want : most;
    Q.splits = (int)(want < 1 ? 1 : (want < 64 ? want : 64));
    if (S.fused) {
        const int waves = a->dim <= 64 ? 4 : 2;
        Q.row_blocks = 1;
        Q.items = a->batch * a->kv_heads;
        want = 512 / Q.items;   // two workgroups a compute unit: a third would wait for them
        most = a->passages * ((a->len + 31) / 32) / (4 * waves);
        want = want < most ? want : most;
        Q.splits = (int)(want < 1 ? 1 : (want < 64 ? want : 64));
    }
    AttendPlan& K = S.kv;
    K.row_blocks = 1;
    K.by_head = K.row_count > 64;
    K.items = a->batch * a->kv_heads * ((a->passages * ((a->len + 31) / 32) + 3) / 4);
    want = (512 + K.items - 1) / K.items;
    most = (K.row_count + 63) / 64 / 2;
    want = want < most ? want : most;
    K.splits = (int)(want < 1 ? 1 : (want < 64 ? want : 64));
    S.all_q = a->batch * a->rows * a->heads * a->dim;
    S.all_k = a->batch * a->passages * a->len * a->kv_heads * a->dim;
    S.stats = 0;
    S.part = round_up(a->batch * a->kv_heads * Q.pad_rows * (int64_t)sizeof(RowStat), 256);
    const int64_t pq = Q.splits > 1 ? Q.splits * S.all_q * 4 : 0, pk = !S.fused && K.splits > 1 ? K.splits * 2 * S.all_k * 4 : 0;
    S.total = S.part + round_up(pq > pk ? pq : pk, 256);
    return S;
}

extern "C" int64_t artread_attend_grad_workspace(const artread_attend_t* a) {
    const int rc = check_attend(a);
    return rc ? rc : grad_shape(a).total;
}

template <typename T>
static void launch_sum(const float* part, int64_t stride, int splits, void* out, int64_t n, hipStream_t st) {
    hipLaunchKernelGGL((attend_sum_kernel<T>), dim3(grid_of((n + 1023) / 1024)), dim3(256), 0, st, part, stride, splits,
                       (T*)out, n);
}

template <typename T, int DP>
static void launch_attend_grad(const artread_attend_t* a, const artread_attend_grads_t* g, const GradShape& S, void* ws,
                               hipStream_t st) {
    RowStat* stats = (RowStat*)((char*)ws + S.stats);
    float* part = (float*)((char*)ws + S.part);
    const int64_t rows = a->batch * a->kv_heads * S.q.pad_rows;
    hipLaunchKernelGGL((attend_delta_kernel<T>), dim3(grid_of((rows + 15) / 16)), dim3(256), 0, st, *a, *g, S.q, rows, stats);
    if (S.fused) {
        const dim3 grid = grid2(S.q.items * S.q.splits);
        constexpr int NW = DP == 64 ? 4 : 2;
#define GRADS(RB, PACK) \
    hipLaunchKernelGGL((attend_grad_stream_kernel<T, DP, RB, NW, PACK>), grid, dim3(64 * NW), 0, st, *a, *g, S.q, stats, part)
        if constexpr (DP == 64) {
            if (S.q.row_count > 32) {
                if (S.q.pack) GRADS(2, true);
                else GRADS(2, false);
            }
        }
        if (S.q.row_count <= 32) {
            if (S.q.pack) GRADS(1, true);
            else GRADS(1, false);
        }
#undef GRADS
        if (S.q.splits > 1) launch_sum<T>(part, S.all_q, S.q.splits, g->grad_q, S.all_q, st);
        return;
    }
    const dim3 gq = grid2(S.q.items * S.q.splits);
    if constexpr (DP == 128)   // 33 to 64 rows; at 64 columns they are the one walk's
        if (S.narrow) hipLaunchKernelGGL((attend_grad_q_kernel<T, DP, 1, 1>), gq, dim3(64), 0, st, *a, *g, S.q, stats, part);
    if (!S.narrow) hipLaunchKernelGGL((attend_grad_q_kernel<T, DP, 4, 2>), gq, dim3(256), 0, st, *a, *g, S.q, stats, part);
    if (S.q.splits > 1) launch_sum<T>(part, S.all_q, S.q.splits, g->grad_q, S.all_q, st);
    hipLaunchKernelGGL((attend_grad_kv_kernel<T, DP>), grid2(S.kv.items * S.kv.splits), dim3(256), 0, st, *a, *g,
                       S.kv, stats, part);
    if (S.kv.splits > 1) {
        launch_sum<T>(part, 2 * S.all_k, S.kv.splits, g->grad_k, S.all_k, st);
        launch_sum<T>(part + S.all_k, 2 * S.all_k, S.kv.splits, g->grad_v, S.all_k, st);
    }
}

extern "C" int artread_attend_grad(int device, const artread_attend_t* a, const artread_attend_grads_t* gr,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_attend_call(a);
    if (rc) return rc;
    READ_ARG(gr && a->lse && gr->grad_out && gr->grad_q && gr->grad_k && gr->grad_v, "a pointer is NULL");
    const int64_t strides[3] = {gr->g_batch, gr->g_row, gr->g_head};
    for (int i = 0; i < 3; ++i)
        READ_ARG(strides[i] >= 0 && strides[i] % 8 == 0 && strides[i] < kStrideLimit,
                 "strides must be multiples of 8 in [0, 2^40)");
    READ_ARG(tile_fits(gr->g_row, gr->g_head, a->heads / a->kv_heads),
             "row strides must be below 2^24, the query heads that share a key head within 2^29 elements");
    READ_ARG(aligned(gr->grad_out, 16) && aligned(gr->grad_q, 16) && aligned(gr->grad_k, 16) && aligned(gr->grad_v, 16),
             "gradients must be 16-byte aligned");
    const GradShape S = grad_shape(a);
    READ_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= S.total,
             "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)S.total);
    ReadDeviceGuard g(device);
    READ_HIP(g.err);
    hipStream_t st = (hipStream_t)stream;
    a = &S.args;
    if (a->dtype == ARTREAD_F16) {
        if (a->dim <= 64) launch_attend_grad<f16, 64>(a, gr, S, workspace, st);
        else launch_attend_grad<f16, 128>(a, gr, S, workspace, st);
    } else {
        if (a->dim <= 64) launch_attend_grad<bf16, 64>(a, gr, S, workspace, st);
        else launch_attend_grad<bf16, 128>(a, gr, S, workspace, st);
    }
    READ_HIP(hipGetLastError());
    return 0;
}
