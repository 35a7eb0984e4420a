/* Refusals and error paths of the 8-bit projections, the append with norms and the
 * attention over a shared prefix, on the HIP runtime of host_paths_check.c (no GPU:
 * kernels are counted, not run). */
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

static void append_norm(void) {
    static _Alignas(64) float gain[2][HD];
    const tl_paged_cache c = cache();
    const int64_t w = (HEADS + 2 * KV) * HD, qw = HEADS * HD;
    const int bad = TL_ERR_BAD_DESCRIPTOR;
#define AN(rows, g, k, eps) tl_paged_append_norm(H, &c, qkv, w, TL_F32, rows, HEADS, seq, pos, cs, sn, 64, g, k, eps, q, qw)
    expect("norm", AN(4, gain[0], gain[1], 1e-5), TL_OK, 1);
    expect("norm, no rows", AN(0, gain[0], gain[1], 1e-5), TL_OK, 0);
    expect("norm of q only", AN(4, gain[0], NULL, 0.0), TL_OK, 1);
    expect("norm of k only", AN(4, NULL, gain[1], 1e-6), TL_OK, 1);
    expect("no norm", AN(4, NULL, NULL, -1.0), TL_OK, 1);
    expect("misaligned q gain", AN(4, gain[0] + 1, gain[1], 1e-5), bad, 0);
    expect("misaligned k gain", AN(4, gain[0], gain[1] + 2, 1e-5), bad, 0);
    expect("negative eps", AN(4, gain[0], gain[1], -1e-5), bad, 0);
    expect("NaN eps", AN(4, gain[0], gain[1], 0.0 / 0.0), bad, 0);
    expect("infinite eps", AN(4, gain[0], gain[1], 1.0 / 0.0), bad, 0);
    expect("norm: negative rows", AN(-1, gain[0], gain[1], 1e-5), bad, 0);
    expect("norm async", tl_paged_append_norm_async(H, NULL, &c, qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64, gain[0],
                                                    gain[1], 1e-5, q, qw, NULL), TL_OK, 1);
    expect("norm async: eps", tl_paged_append_norm_async(H, NULL, &c, qkv, w, TL_F32, 4, HEADS, seq, pos, cs, sn, 64,
                                                         gain[0], gain[1], -1.0, q, qw, NULL), bad, 0);
    queued = 0;
}

static void shared(void) {
    tl_paged_cache c = cache();
    const int64_t qw = HEADS * HD;
    const int bad = TL_ERR_BAD_DESCRIPTOR;
    int64_t need = -1, own = -1;
#define SH(rows, ps, len) tl_paged_attention_shared(H, &c, q, qw, TL_F32, rows, HEADS, seq, pos, ps, len, 0.125f, out, qw)
    expect("shared", SH(4, 0, 20), TL_OK, 2);
    expect("shared, the whole table", SH(4, SEQS - 1, PAGE * MAXP), TL_OK, 2);
    expect("shared, no prefix", SH(4, 0, 0), TL_OK, 1);
    expect("shared, no prefix of any sequence", SH(4, 99, 0), TL_OK, 1);
    expect("shared, no rows", SH(0, 0, 20), TL_OK, 0);
    expect("prefix past the table", SH(4, 0, PAGE * MAXP + 1), bad, 0);
    expect("negative prefix", SH(4, 0, -1), bad, 0);
    expect("prefix of no sequence", SH(4, SEQS, 20), bad, 0);
    expect("prefix of a negative sequence", SH(4, -1, 20), bad, 0);
    expect("shared: negative rows", SH(-1, 0, 20), bad, 0);
    expect("shared: null q", tl_paged_attention_shared(H, &c, NULL, qw, TL_F32, 4, HEADS, seq, pos, 0, 20, 1, out, qw), bad, 0);
    expect("shared: heads", tl_paged_attention_shared(H, &c, q, qw, TL_F32, 4, 7, seq, pos, 0, 20, 1, out, qw), bad, 0);
    expect("shared: out a row on", tl_paged_attention_shared(H, &c, q, qw, TL_F32, 3, HEADS, seq, pos, 0, 20, 1, &q[1][0], qw), bad, 0);
    expect("shared: out is q", tl_paged_attention_shared(H, &c, q, qw, TL_F32, 4, HEADS, seq, pos, 0, 20, 1, q, qw), TL_OK, 2);
    expect("shared scratch", tl_paged_attention_shared_scratch(H, &c, 4, HEADS, 20, &need), TL_OK, 0);
    expect("scratch", tl_paged_attention_scratch(H, &c, 4, HEADS, &own), TL_OK, 0);
    checks++;
    wrong += need < own + 4 * HEADS * (HD + 2) * 4;
    expect("shared scratch, none", tl_paged_attention_shared_scratch(H, &c, 4, HEADS, 0, &need), TL_OK, 0);
    checks++;
    wrong += need != own;
    expect("shared scratch null", tl_paged_attention_shared_scratch(H, &c, 4, HEADS, 20, NULL), bad, 0);
    expect("shared scratch prefix", tl_paged_attention_shared_scratch(H, &c, 4, HEADS, 99, &need), bad, 0);
    expect("shared scratch cache", tl_paged_attention_shared_scratch(H, NULL, 4, HEADS, 20, &need), bad, 0);
    expect("shared scratch rows", tl_paged_attention_shared_scratch(H, &c, -1, HEADS, 20, &need), bad, 0);
    tl_paged_cache one = cache();   /* 2^30 query heads */
    one.max_pages = 1;
    expect("too many heads", tl_paged_attention_shared_scratch(H, &one, 1 << 15, 1 << 15, 5, &need), TL_ERR_UNSUPPORTED, 0);
    expect("shared scratch", tl_paged_attention_shared_scratch(H, &c, 4, HEADS, 20, &need), TL_OK, 0);
    char* s = aligned_alloc(64, (size_t)(need + 127) / 64 * 64);
#define AS2(scr, n) tl_paged_attention_shared_async(H, NULL, &c, q, qw, TL_F32, 4, HEADS, seq, pos, 0, 20, 1, out, qw, scr, n, NULL, NULL)
    expect("shared async", AS2(s, need), TL_OK, 2);
    expect("shared async, no scratch", AS2(NULL, need), bad, 0);
    expect("shared async, short scratch", AS2(s, need - 1), bad, 0);
    expect("shared async, misaligned scratch", AS2(s + 8, need), bad, 0);
    queued = 0;
    free(s);
    /* a launch that fails */
    for (long f = 1; f <= 2; f++) {
        fail_at = f;
        ops = 0;
        const int r = SH(4, 0, 20);
        fail_at = 0;
        checks++;
        wrong += r != TL_ERR_INTERNAL || queued != 0;
        ops = 0;
        expect("after a failed launch", SH(4, 0, 20), TL_OK, 2);
    }
}

static void linear_w8(void) {
    static _Alignas(64) int8_t w[2][33 * 77];
    static _Alignas(64) float x[4][80], y[4][40], r[4][40], sc[2][33];
    const int bad = TL_ERR_BAD_DESCRIPTOR, uns = TL_ERR_UNSUPPORTED;
    int64_t size = 0, pair = 0, need = -1;
    expect("packed bytes", tl_w8_packed_bytes(H, 33, 77, 0, &size), TL_OK, 0);
    expect("packed bytes of a pair", tl_w8_packed_bytes(H, 33, 77, 1, &pair), TL_OK, 0);
    checks++;
    wrong += size <= 33 * 77 || pair != 2 * size;
    expect("packed bytes null", tl_w8_packed_bytes(H, 33, 77, 0, NULL), bad, 0);
    expect("packed bytes n", tl_w8_packed_bytes(H, 0, 77, 0, &size), bad, 0);
    expect("packed bytes k", tl_w8_packed_bytes(H, 33, 0, 0, &size), bad, 0);
    expect("packed bytes, long k", tl_w8_packed_bytes(H, 33, (1 << 17) + 1, 0, &need), uns, 0);
    expect("packed bytes, many", tl_w8_packed_bytes(H, 1 << 24, 1 << 12, 0, &need), bad, 0);
    char* wp = aligned_alloc(64, (size_t)(pair + 63) / 64 * 64);
    expect("pack", tl_pack_w8(H, w[0], sc[0], NULL, NULL, 33, 77, wp), TL_OK, 1);
    expect("pack a pair", tl_pack_w8(H, w[0], sc[0], w[1], sc[1], 33, 77, wp), TL_OK, 1);
    expect("pack null", tl_pack_w8(H, NULL, sc[0], NULL, NULL, 33, 77, wp), bad, 0);
    expect("pack null scales", tl_pack_w8(H, w[0], NULL, NULL, NULL, 33, 77, wp), bad, 0);
    expect("pack null out", tl_pack_w8(H, w[0], sc[0], NULL, NULL, 33, 77, NULL), bad, 0);
    expect("pack misaligned", tl_pack_w8(H, w[0], sc[0], NULL, NULL, 33, 77, wp + 8), bad, 0);
    expect("pack half a pair", tl_pack_w8(H, w[0], sc[0], w[1], NULL, 33, 77, wp), bad, 0);
    expect("pack half a pair", tl_pack_w8(H, w[0], sc[0], NULL, sc[1], 33, 77, wp), bad, 0);
    expect("pack misaligned scales", tl_pack_w8(H, w[0], (float*)((char*)sc + 2), NULL, NULL, 33, 77, wp), bad, 0);
#define W8(xx, xs, act, m, p, gated, n, k, rr, rs, yy, ys) tl_linear_w8(H, xx, xs, act, m, p, gated, n, k, rr, rs, yy, ys)
    expect("w8", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, r, 40, y, 40), TL_OK, 1);
    expect("w8 gated", W8(x, 80, TL_F32, 4, wp, 1, 33, 77, NULL, 0, y, 40), TL_OK, 1);
    expect("w8 odd rows", W8(&x[0][1], 77, TL_F32, 4, wp, 0, 33, 77, NULL, 0, &y[0][1], 33), TL_OK, 1);
    expect("w8 onto the residual", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, y, 40, y, 40), TL_OK, 1);
    expect("w8 no rows", W8(x, 80, TL_F32, 0, wp, 0, 33, 77, NULL, 0, y, 40), TL_OK, 0);
    expect("w8 gated with a residual", W8(x, 80, TL_F32, 4, wp, 1, 33, 77, r, 40, y, 40), bad, 0);
    expect("w8 int8 rows", W8(x, 80, TL_I8, 4, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 negative rows", W8(x, 80, TL_F32, -1, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 too many rows", W8(x, 80, TL_F32, (1 << 17) + 1, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 too many results", W8(x, 80, TL_F32, 1 << 17, wp, 0, 1 << 21, 77, NULL, 0, y, 1 << 21), uns, 0);
    expect("w8 no columns", W8(x, 80, TL_F32, 4, wp, 0, 0, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 k 0", W8(x, 80, TL_F32, 4, wp, 0, 33, 0, NULL, 0, y, 40), bad, 0);
    expect("w8 null x", W8(NULL, 80, TL_F32, 4, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 null y", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, NULL, 0, NULL, 40), bad, 0);
    expect("w8 null weights", W8(x, 80, TL_F32, 4, NULL, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 misaligned weights", W8(x, 80, TL_F32, 4, wp + 4, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 overlapping x", W8(x, 76, TL_F32, 4, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 overlapping y", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, NULL, 0, y, 32), bad, 0);
    expect("w8 overlapping residual", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, r, 32, y, 40), bad, 0);
    expect("w8 misaligned x", W8((char*)x + 2, 79, TL_F32, 4, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 misaligned y", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, NULL, 0, (char*)y + 1, 39), bad, 0);
    expect("w8 misaligned 16-bit x", W8((char*)x + 1, 79, TL_BF16, 4, wp, 0, 33, 77, NULL, 0, y, 40), bad, 0);
    expect("w8 y on x", W8(x, 80, TL_F32, 4, wp, 0, 33, 77, NULL, 0, x, 80), bad, 0);
    expect("w8 y a row on from the residual", W8(x, 80, TL_F32, 3, wp, 0, 33, 77, &y[0][0], 40, &y[1][0], 40), bad, 0);
    expect("w8 scratch of few rows", tl_linear_w8_scratch(H, 4, 77, &need), TL_OK, 0);
    checks++;
    wrong += need != 0;
    expect("w8 scratch null", tl_linear_w8_scratch(H, 4, 77, NULL), bad, 0);
    expect("w8 scratch rows", tl_linear_w8_scratch(H, -4, 77, &need), bad, 0);
    expect("w8 scratch k", tl_linear_w8_scratch(H, 4, (1 << 17) + 1, &need), bad, 0);
    static _Alignas(64) float big[400][80], bout[400][40];
    for (int m = 40; m <= 400; m += 360) {
        expect("w8 scratch", tl_linear_w8_scratch(H, m, 77, &need), TL_OK, 0);
        char* s = aligned_alloc(64, (size_t)(need + 127) / 64 * 64);
#define AW8(scr, n) tl_linear_w8_async(H, NULL, big, 80, TL_F32, m, wp, 0, 33, 77, NULL, 0, bout, 40, scr, n)
        expect("w8 async", AW8(s, need), TL_OK, 2);
        expect("w8 async, no scratch", AW8(NULL, need), bad, 0);
        expect("w8 async, short scratch", AW8(s, need - 1), bad, 0);
        expect("w8 async, misaligned scratch", AW8(s + 4, need), bad, 0);
        queued = 0;
        free(s);
    }
    for (long f = 1; f <= 2; f++) {   /* a launch that fails */
        fail_at = f;
        ops = 0;
        const int got = W8(big, 80, TL_F32, 40, wp, 0, 33, 77, NULL, 0, bout, 40);
        fail_at = 0;
        checks++;
        wrong += got != TL_ERR_INTERNAL || queued != 0;
        ops = 0;
        expect("after a failed launch", W8(big, 80, TL_F32, 40, wp, 0, 33, 77, NULL, 0, bout, 40), TL_OK, 2);
    }
    expect("null handle", tl_linear_w8_scratch(NULL, 4, 77, &need), bad, 0);
    free(wp);
}

int main(void) {
    H = make(1024, 4);
    ops = 0;
    append_norm();
    shared();
    linear_w8();
    tl_destroy(H);
    printf("%d checks, %d wrong\n", checks, wrong);
    return wrong > 255 ? 255 : wrong;
}
