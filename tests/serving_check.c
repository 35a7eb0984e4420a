/* Refusals and error paths of the serving operators, on the HIP runtime of
 * host_paths_check.c (no GPU: kernels are counted, not run).  Every call that
 * an argument rules out returns its status and a message, launches nothing and
 * leaves the handle usable; a completing call whose launch fails returns an
 * error with nothing left queued. */
#define main host_paths_main
#include "host_paths_check.c"
#undef main

static int checks, wrong;
static tl_handle* H;

static void expect(const char* what, int got, int want, long launches) {
    checks++;
    const int ok = got == want && ops == launches && (want == TL_OK || tl_last_error(H)[0]);
    if (!ok) {
        wrong++;
        printf("%s: status %d, want %d; %ld launches, want %ld; \"%s\"\n", what, got, want, ops, launches, tl_last_error(H));
    }
    ops = 0;
}

enum { HD = 64, KV = 2, HEADS = 8, PAGE = 16, PAGES = 6, SEQS = 3, MAXP = 2 };
static _Alignas(64) int8_t k_pages[PAGES * KV * PAGE * HD], v_pages[sizeof k_pages];
static _Alignas(64) float ks[KV], vs[KV], qkv[4][(HEADS + 2 * KV) * HD], q[4][HEADS * HD], out[4][HEADS * HD];
static _Alignas(64) float cs[64 * HD], sn[64 * HD];
static int32_t table[SEQS * MAXP], seq[4], pos[4];

static tl_paged_cache cache(void) {
    const tl_paged_cache c = {k_pages, v_pages, ks, vs, table, MAXP, KV * PAGE * HD, TL_I8, PAGES, PAGE, KV, HD, SEQS, MAXP};
    return c;
}
static int append(const tl_paged_cache* c) {
    return tl_paged_append(H, c, qkv, (HEADS + 2 * KV) * HD, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, HEADS * HD);
}
static int attend(const tl_paged_cache* c) {
    return tl_paged_attention(H, c, q, HEADS * HD, TL_F32, 4, HEADS, seq, pos, 0.125f, out, HEADS * HD);
}
static void both(const char* what, tl_paged_cache c, int want) {
    expect(what, append(&c), want, 0);
    expect(what, attend(&c), want, 0);
}

static void paged(void) {
    tl_paged_cache c = cache();
    const int64_t w = (HEADS + 2 * KV) * HD, qw = HEADS * HD;
    int64_t need = -1;
    expect("append", append(&c), TL_OK, 1);
    expect("scratch", tl_paged_attention_scratch(H, &c, 4, HEADS, &need), TL_OK, 0);
    expect("attention", attend(&c), TL_OK, 1);
    expect("no rows", tl_paged_append(H, &c, qkv, w, TL_F32, 0, HEADS, NULL, NULL, cs, sn, 64, q, qw), TL_OK, 0);
    expect("no rows", tl_paged_attention(H, &c, q, qw, TL_F32, 0, HEADS, NULL, NULL, 1, out, qw), TL_OK, 0);
    expect("no queries", tl_paged_append(H, &c, qkv, 2 * KV * HD, TL_F32, 4, 0, seq, pos, cs, sn, 64, NULL, 0), TL_OK, 1);
    expect("in place", tl_paged_append(H, &c, qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, qkv, w), TL_OK, 1);
#define WITH(what, change, want) do { tl_paged_cache x = cache(); change; both(what, x, want); } while (0)
    WITH("null k", x.k = NULL, TL_ERR_BAD_DESCRIPTOR);
    WITH("null table", x.table = NULL, TL_ERR_BAD_DESCRIPTOR);
    WITH("no scales", x.k_scale = NULL, TL_ERR_BAD_DESCRIPTOR);
    WITH("float32 cache", x.dtype = TL_F32, TL_ERR_BAD_DESCRIPTOR);
    WITH("type", x.dtype = 9, TL_ERR_BAD_DESCRIPTOR);
    WITH("head_dim", x.head_dim = 96, TL_ERR_UNSUPPORTED);
    WITH("page 4", x.page_size = 4, TL_ERR_UNSUPPORTED);
    WITH("page 24", x.page_size = 24, TL_ERR_UNSUPPORTED);
    WITH("page 2048", x.page_size = 2048, TL_ERR_UNSUPPORTED);
    WITH("page 0", x.page_size = 0, TL_ERR_UNSUPPORTED);
    WITH("no pages", x.n_pages = 0, TL_ERR_BAD_DESCRIPTOR);
    WITH("no KV heads", x.n_kv_heads = 0, TL_ERR_BAD_DESCRIPTOR);
    WITH("no sequences", x.n_seqs = 0, TL_ERR_BAD_DESCRIPTOR);
    WITH("no entries", x.max_pages = 0, TL_ERR_BAD_DESCRIPTOR);
    WITH("too long", (x.max_pages = 1 << 27, x.table_stride = 1 << 27), TL_ERR_BAD_DESCRIPTOR);
    WITH("table_stride", x.table_stride = MAXP - 1, TL_ERR_BAD_DESCRIPTOR);
    WITH("misaligned k", x.k = k_pages + 8, TL_ERR_BAD_DESCRIPTOR);
    WITH("misaligned v", x.v = v_pages + 1, TL_ERR_BAD_DESCRIPTOR);
    WITH("short page_stride", x.page_stride -= 16, TL_ERR_BAD_DESCRIPTOR);
    WITH("odd page_stride", x.page_stride += 8, TL_ERR_BAD_DESCRIPTOR);
    WITH("huge page_stride", x.page_stride = (int64_t)1 << 32, TL_ERR_BAD_DESCRIPTOR);
    expect("null cache", append(NULL), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("null cache", attend(NULL), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("null cache", tl_paged_attention_scratch(H, NULL, 4, HEADS, &need), TL_ERR_BAD_DESCRIPTOR, 0);
#define APP(what, ...) expect("append: " what, tl_paged_append(H, &c, __VA_ARGS__), TL_ERR_BAD_DESCRIPTOR, 0)
    APP("null qkv", NULL, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("int8 rows", qkv, w, TL_I8, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("too many rows", qkv, w, TL_F32, 1 << 24, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("negative rows", qkv, w, TL_F32, -1, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("negative heads", qkv, w, TL_F32, 4, -1, seq, pos, cs, sn, 64, q, qw);
    APP("null pos", qkv, w, TL_F32, 4, HEADS, seq, NULL, cs, sn, 64, q, qw);
    APP("null cos", qkv, w, TL_F32, 4, HEADS, seq, pos, NULL, sn, 64, q, qw);
    APP("no table rows", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 0, q, qw);
    APP("misaligned sin", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn + 1, 64, q, qw);
    APP("overlapping rows", qkv, w - 4, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("odd stride", qkv, w + 1, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("odd 16-bit stride", qkv, w + 4, TL_F16, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("misaligned rows", &qkv[0][1], w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw);
    APP("misaligned q_out", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, &q[0][2], qw);
    APP("short q_stride", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw - 4);
    APP("in place, another stride", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, qkv, qw);
    APP("q_out on k", qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, &qkv[0][2 * HD], w);
    APP("q_out a row on", qkv, w, TL_F32, 3, HEADS, seq, pos, cs, sn, 64, &qkv[1][0], w);
#define ATT(what, ...) expect("attention: " what, tl_paged_attention(H, &c, __VA_ARGS__), TL_ERR_BAD_DESCRIPTOR, 0)
    ATT("null q", NULL, qw, TL_F32, 4, HEADS, seq, pos, 1, out, qw);
    ATT("null out", q, qw, TL_F32, 4, HEADS, seq, pos, 1, NULL, qw);
    ATT("int8 rows", q, qw, TL_I8, 4, HEADS, seq, pos, 1, out, qw);
    ATT("no heads", q, qw, TL_F32, 4, 0, seq, pos, 1, out, qw);
    ATT("7 heads on 2", q, qw, TL_F32, 4, 7, seq, pos, 1, out, qw);
    ATT("null pos", q, qw, TL_F32, 4, HEADS, seq, NULL, 1, out, qw);
    ATT("negative rows", q, qw, TL_F32, -4, HEADS, seq, pos, 1, out, qw);
    ATT("short stride", q, qw - 4, TL_F32, 4, HEADS, seq, pos, 1, out, qw);
    ATT("misaligned out", q, qw, TL_F32, 4, HEADS, seq, pos, 1, &out[0][1], qw);
    ATT("out a row on", q, qw, TL_F32, 3, HEADS, seq, pos, 1, &q[1][0], qw);
    ATT("out on q, another stride", q, qw, TL_F32, 2, HEADS, seq, pos, 1, q, qw + 4);
    expect("out is q", tl_paged_attention(H, &c, q, qw, TL_F32, 4, HEADS, seq, pos, 1, q, qw), TL_OK, 1);
    tl_paged_cache deep = cache();
    deep.max_pages = 1 << 26;   /* 2^30 positions: 2^22 tiles */
    deep.table_stride = 1 << 26;
    expect("too many tiles", tl_paged_attention(H, &deep, q, qw, TL_F32, 300, HEADS, seq, pos, 1, out, qw), TL_ERR_UNSUPPORTED, 0);
    expect("scratch: null", tl_paged_attention_scratch(H, &c, 4, HEADS, NULL), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("scratch: heads", tl_paged_attention_scratch(H, &c, 4, 3, &need), TL_ERR_BAD_DESCRIPTOR, 0);

    /* the form on the caller's stream: a long cache needs scratch */
    tl_paged_cache l = cache();
    static int32_t wide[SEQS * 512];
    l.table = wide;
    l.table_stride = l.max_pages = 512;
    expect("long scratch", tl_paged_attention_scratch(H, &l, 1, HEADS, &need), TL_OK, 0);
    checks++;
    wrong += need <= 0;
    void* s = aligned_alloc(64, (size_t)(need + 127) / 64 * 64);
#define ASYNC(scr, n) tl_paged_attention_async(H, NULL, &l, q, qw, TL_F32, 1, HEADS, seq, pos, 1, out, qw, scr, n, NULL, NULL)
    expect("async", ASYNC(s, need), TL_OK, 2);
    expect("async, no scratch", ASYNC(NULL, need), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("async, short scratch", ASYNC(s, need - 1), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("async, misaligned scratch", ASYNC((char*)s + 4, need), TL_ERR_BAD_DESCRIPTOR, 0);
    expect("async append", tl_paged_append_async(H, NULL, &c, qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, q, qw, NULL),
           TL_OK, 1);
    free(s);
    queued = 0;   /* what the async calls queued */

    /* a launch that fails */
    for (long f = 1; f <= 2; f++) {
        fail_at = f;
        ops = 0;
        const int r = tl_paged_attention(H, &l, q, qw, TL_F32, 1, HEADS, seq, pos, 1, out, qw);
        fail_at = 0;
        checks++;
        wrong += r != TL_ERR_INTERNAL || queued != 0;
        ops = 0;
        expect("after a failed launch", tl_paged_attention(H, &l, q, qw, TL_F32, 1, HEADS, seq, pos, 1, out, qw), TL_OK, 2);
    }
    expect("null handle", tl_paged_attention_scratch(NULL, &c, 1, HEADS, &need), TL_ERR_BAD_DESCRIPTOR, 0);
}

static void linear_w4(void) {
    static _Alignas(64) uint8_t w[32 * 128];
    static _Alignas(64) float x[4][256], y[4][32], r[4][32], sc[32 * 8], wf[32 * 256];
    const int bad = TL_ERR_BAD_DESCRIPTOR, uns = TL_ERR_UNSUPPORTED;
    int64_t need = 0, size = 0;
    expect("packed bytes", tl_w4_packed_bytes(H, 32, 256, 64, TL_F32, &size), TL_OK, 0);
    void* wp = aligned_alloc(64, (size_t)(size + 63) / 64 * 64);
    expect("pack", tl_pack_w4(H, w, sc, TL_F32, 64, 32, 256, wp), TL_OK, 1);
    expect("pack null", tl_pack_w4(H, NULL, sc, TL_F32, 64, 32, 256, wp), bad, 0);
    expect("pack null out", tl_pack_w4(H, w, sc, TL_F32, 64, 32, 256, NULL), bad, 0);
    expect("pack misaligned", tl_pack_w4(H, w, sc, TL_F32, 64, 32, 256, (char*)wp + 8), bad, 0);
    expect("pack misaligned q", tl_pack_w4(H, w + 2, sc, TL_F32, 64, 32, 256, wp), bad, 0);
    expect("pack misaligned scales", tl_pack_w4(H, w, (char*)sc + 2, TL_F32, 64, 32, 256, wp), bad, 0);
    expect("pack group", tl_pack_w4(H, w, sc, TL_F32, 48, 32, 256, wp), uns, 0);
    expect("pack too many rows", tl_pack_w4(H, w, sc, TL_F32, 64, (1 << 24) + 1, 256, wp), bad, 0);
    expect("pack too many weights", tl_pack_w4(H, w, sc, TL_F32, 64, 1 << 24, 4096, wp), bad, 0);
    expect("pack no rows", tl_pack_w4(H, w, sc, TL_F32, 64, 0, 256, wp), bad, 0);
    expect("pack scale type", tl_pack_w4(H, w, sc, TL_I8, 64, 32, 256, wp), bad, 0);
    expect("packed bytes null", tl_w4_packed_bytes(H, 32, 256, 64, TL_F32, NULL), bad, 0);
    expect("packed bytes group", tl_w4_packed_bytes(H, 32, 256, 16, TL_F32, &size), uns, 0);
#define W4(xx, xs, act, m, p, st, grp, n, k, rr, rs, yy, ys) tl_linear_w4(H, xx, xs, act, m, p, st, grp, n, k, rr, rs, yy, ys)
    expect("w4", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, r, 32, y, 32), TL_OK, 1);
    expect("no rows", W4(x, 256, TL_F32, 0, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), TL_OK, 0);
    expect("int8 rows", W4(x, 256, TL_I8, 4, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("scale type", W4(x, 256, TL_F32, 4, wp, TL_I8, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("negative rows", W4(x, 256, TL_F32, -1, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("too many rows", W4(x, 256, TL_F32, (1 << 17) + 1, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("no columns", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 0, 256, NULL, 0, y, 32), bad, 0);
    expect("k 0", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 0, NULL, 0, y, 32), bad, 0);
    expect("k 200", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 200, NULL, 0, y, 32), uns, 0);
    expect("group 16", W4(x, 256, TL_F32, 4, wp, TL_F32, 16, 32, 256, NULL, 0, y, 32), uns, 0);
    expect("group 0", W4(x, 256, TL_F32, 4, wp, TL_F32, 0, 32, 256, NULL, 0, y, 32), uns, 0);
    expect("many groups", W4(x, 65536, TL_F32, 4, wp, TL_F32, 32, 32, 65536, NULL, 0, y, 32), uns, 0);
    expect("null weights", W4(x, 256, TL_F32, 4, NULL, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("misaligned weights", W4(x, 256, TL_F32, 4, (char*)wp + 8, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("null x", W4(NULL, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("null y", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, NULL, 32), bad, 0);
    expect("short x", W4(x, 252, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("odd x", W4(x, 257, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("misaligned x", W4(&x[0][1], 256, TL_F32, 3, wp, TL_F32, 64, 32, 256, NULL, 0, y, 32), bad, 0);
    expect("short y", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, y, 31), bad, 0);
    expect("misaligned y", W4(x, 256, TL_F32, 3, wp, TL_F32, 64, 32, 256, NULL, 0, (char*)y + 2, 32), bad, 0);
    expect("short residual", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, r, 31, y, 32), bad, 0);
    expect("y on x", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, NULL, 0, x, 256), bad, 0);
    expect("y in x's rows", W4(x, 256, TL_F32, 2, wp, TL_F32, 64, 32, 128, NULL, 0, &x[0][128], 256), TL_OK, 1);
    expect("y and x meet", W4(x, 256, TL_F32, 2, wp, TL_F32, 64, 32, 128, NULL, 0, &x[0][127], 256), bad, 0);
    expect("residual is y", W4(x, 256, TL_F32, 4, wp, TL_F32, 64, 32, 256, y, 32, y, 32), TL_OK, 1);
    expect("residual shifted", W4(x, 256, TL_F32, 2, wp, TL_F32, 64, 32, 256, (char*)y + 4, 32, y, 32), bad, 0);
    expect("scratch null", tl_linear_w4_scratch(H, 4, 256, NULL), bad, 0);
    expect("scratch rows", tl_linear_w4_scratch(H, -4, 256, &need), bad, 0);
    expect("quantize", tl_quantize_w4_rows(H, wf, 32, 256, 64, TL_F32, w, sc), TL_OK, 1);
    expect("quantize no rows", tl_quantize_w4_rows(H, wf, 0, 256, 64, TL_F32, w, sc), TL_OK, 0);
    expect("quantize null", tl_quantize_w4_rows(H, NULL, 32, 256, 64, TL_F32, w, sc), bad, 0);
    expect("quantize group", tl_quantize_w4_rows(H, wf, 32, 256, 40, TL_F32, w, sc), uns, 0);
    expect("quantize type", tl_quantize_w4_rows(H, wf, 32, 256, 64, TL_I8, w, sc), bad, 0);
    expect("quantize misaligned", tl_quantize_w4_rows(H, wf + 1, 31, 256, 64, TL_F32, w, sc), bad, 0);
    /* the form on the caller's stream */
    static _Alignas(64) float big[40][256], out[40][32];
    expect("w4 scratch", tl_linear_w4_scratch(H, 40, 256, &need), TL_OK, 0);
    char* s = aligned_alloc(64, (size_t)(need + 127) / 64 * 64);
#define AW(scr, n) tl_linear_w4_async(H, NULL, big, 256, TL_F32, 40, wp, TL_F32, 64, 32, 256, NULL, 0, out, 32, scr, n)
    expect("async", AW(s, need), TL_OK, 2);
    expect("async, no scratch", AW(NULL, need), bad, 0);
    expect("async, short scratch", AW(s, need - 1), bad, 0);
    expect("async, misaligned scratch", AW(s + 4, need), bad, 0);
    queued = 0;
    free(s);
    free(wp);
}

static void logprobs(void) {
    static _Alignas(64) float x[2][20000], lp[2], h[2], tl[2][8];
    static int32_t t[2], ids[2][8];
    const int bad = TL_ERR_BAD_DESCRIPTOR;
    int64_t need;
#define LP(x, st, dt, rows, v, t, top, lp, h, ids, tl) tl_token_logprobs(H, x, st, dt, rows, v, t, top, lp, h, ids[0], tl[0])
    expect("logprobs, one part", LP(x, 20000, TL_F32, 2, 5000, t, 8, lp, h, ids, tl), TL_OK, 1);
    expect("logprobs, joined in place", LP(x, 20000, TL_F32, 2, 20000, t, 8, lp, h, ids, tl), TL_OK, 1);
    expect("logprobs, a join", LP(x, 20000, TL_F32, 600, 20000, t, 8, lp, h, ids, tl), TL_OK, 2);
    expect("odd stride", LP((char*)x + 2, 19999, TL_F16, 2, 5000, t, 8, lp, h, ids, tl), TL_OK, 1);
    expect("no rows", LP(x, 20000, TL_F32, 0, 20000, t, 8, lp, h, ids, tl), TL_OK, 0);
    expect("no entropy", LP(x, 20000, TL_F32, 2, 5000, t, 8, lp, NULL, ids, tl), TL_OK, 1);
    expect("no alternatives", tl_token_logprobs(H, x, 20000, TL_F32, 2, 5000, t, 0, lp, h, NULL, NULL), TL_OK, 1);
    expect("null logits", LP(NULL, 20000, TL_F32, 2, 5000, t, 8, lp, h, ids, tl), bad, 0);
    expect("null targets", LP(x, 20000, TL_F32, 2, 5000, NULL, 8, lp, h, ids, tl), bad, 0);
    expect("null logprob", LP(x, 20000, TL_F32, 2, 5000, t, 8, NULL, h, ids, tl), bad, 0);
    expect("null ids", tl_token_logprobs(H, x, 20000, TL_F32, 2, 5000, t, 8, lp, h, NULL, tl[0]), bad, 0);
    expect("int8 logits", LP(x, 20000, TL_I8, 2, 5000, t, 8, lp, h, ids, tl), bad, 0);
    expect("top 33", LP(x, 20000, TL_F32, 2, 5000, t, 33, lp, h, ids, tl), bad, 0);
    expect("top -1", LP(x, 20000, TL_F32, 2, 5000, t, -1, lp, h, ids, tl), bad, 0);
    expect("top above vocab", LP(x, 20000, TL_F32, 2, 7, t, 8, lp, h, ids, tl), bad, 0);
    expect("vocab 0", LP(x, 20000, TL_F32, 2, 0, t, 0, lp, h, ids, tl), bad, 0);
    expect("vocab above 2^28", LP(x, 1 << 30, TL_F32, 2, (1 << 28) + 1, t, 0, lp, h, ids, tl), bad, 0);
    expect("overlapping rows", LP(x, 4999, TL_F32, 2, 5000, t, 8, lp, h, ids, tl), bad, 0);
    expect("misaligned", LP((char*)x + 2, 20000, TL_F32, 2, 5000, t, 8, lp, h, ids, tl), bad, 0);
    expect("too many rows", LP(x, 5000, TL_F32, 1 << 24, 5000, t, 8, lp, h, ids, tl), TL_ERR_UNSUPPORTED, 0);
    expect("too many parts", LP(x, 20000, TL_F32, 1 << 23, 20000, t, 8, lp, h, ids, tl), TL_ERR_UNSUPPORTED, 0);
    expect("negative rows", LP(x, 20000, TL_F32, -2, 5000, t, 8, lp, h, ids, tl), bad, 0);
    expect("scratch", tl_token_logprobs_scratch(H, 2, 20000, 8, &need), TL_OK, 0);
    static char s[4096];
    char* a = (char*)(((uintptr_t)s + 63) & ~(uintptr_t)63);
    checks++;
    wrong += need <= 0 || need > 4000;
#define AS(scr, n) tl_token_logprobs_async(H, NULL, x, 20000, TL_F32, 2, 20000, t, 8, lp, h, ids[0], tl[0], scr, n, NULL, NULL)
    expect("async", AS(a, need), TL_OK, 2);
    expect("async, no scratch", AS(NULL, need), bad, 0);
    expect("async, short scratch", AS(a, need - 1), bad, 0);
    expect("async, misaligned scratch", AS(a + 8, need), bad, 0);
    expect("scratch null", tl_token_logprobs_scratch(H, 2, 20000, 8, NULL), bad, 0);
    expect("scratch top", tl_token_logprobs_scratch(H, 2, 20, 21, &need), bad, 0);
    queued = 0;
}

int main(void) {
    H = make(1024, 4);
    ops = 0;
    paged();
    linear_w4();
    logprobs();
    tl_destroy(H);
    printf("%d checks, %d wrong\n", checks, wrong);
    return wrong > 255 ? 255 : wrong;
}
