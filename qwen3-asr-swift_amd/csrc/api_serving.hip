// extern "C" surface of the serving operators (declared in include/q3asr.h): 8-bit products, paged KV cache, attention over it.
#include "i8.h"
#include "model.h"
#include "paged.h"

#define Q3_API_BEGIN try {
#define Q3_API_END                            \
    q3_set_error("");                         \
    return 0;                                 \
    }                                         \
    catch (const std::exception& e) {         \
        q3_set_error(e.what());               \
        return 1;                             \
    }                                         \
    catch (...) {                             \
        q3_set_error("q3asr: unknown error"); \
        return 2;                             \
    }

namespace {

// A call's device, stream and lock.  The calling thread's current device is put back at the end.
struct Call {
    std::lock_guard<std::mutex> lock;
    int before = -1;
    hipStream_t s;
    bool wait;
    Call(q3asr_model* m, void* stream) : lock(m->call_mutex) {
        HIP_CHECK(hipGetDevice(&before));
        if (before != m->device) HIP_CHECK(hipSetDevice(m->device));
        else before = -1;
        s = stream ? (hipStream_t)stream : m->stream;
        wait = !stream;
    }
    ~Call() { if (before >= 0) (void)hipSetDevice(before); }
    void done() { if (wait) HIP_CHECK(hipStreamSynchronize(s)); }
};

bool aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }

// Strides are counted in values; a buffer has to be addressable with 64 bits and a row's end must not wrap.
constexpr int64_t MAX_LD = (int64_t)1 << 40;
// Rows (and output channels) of one call: a workgroup each stays within what a launch may hold, rounding up to tiles within 32 bits.
constexpr int MAX_ROWS = (1 << 24) - 1;
constexpr int MAX_LD_I8 = 1 << 22;

void check_rows(const char* what, const void* p, int dtype, int64_t ld, int cols) {
    const std::string w(what);
    Q3_REQUIRE(dtype == Q3ASR_F32 || dtype == Q3ASR_BF16, w + ": the type must be Q3ASR_F32 or Q3ASR_BF16");
    Q3_REQUIRE(aligned(p, dtype == Q3ASR_F32 ? 4 : 2), w + ": pointer not aligned to its type");
    Q3_REQUIRE(ld >= cols && ld < MAX_LD, w + ": row stride smaller than a row");
}
void check_i8(const char* what, const int8_t* p, int64_t ld, int cols) {
    const std::string w(what);
    Q3_REQUIRE(aligned(p, 16) && ld % 16 == 0, w + ": 8-bit rows must be aligned to 16 bytes");
    // a tile's rows are addressed by 32-bit byte offsets from its first one
    Q3_REQUIRE(ld >= ((cols + 15) & ~15) && ld <= MAX_LD_I8, w + ": row stride must lie between a row rounded up to 16 and 4194304");
}
int64_t round256(int64_t n) { return (n + 255) & ~255ll; }
int64_t quantized_bytes(int M, int K) { return round256((int64_t)M * ((K + 15) & ~15)) + round256((int64_t)M * 4); }

void check_cache(const q3asr_kv_pages* c, bool workspace) {
    Q3_REQUIRE(c && c->k && c->v && c->table && c->lens && c->refs && c->status, "pages: null argument");
    Q3_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "pages: head_dim must be 64 or 128");
    Q3_REQUIRE(c->page_tokens >= 16 && c->page_tokens <= 256 && (c->page_tokens & (c->page_tokens - 1)) == 0,
               "pages: page_tokens must be a power of two from 16 to 256");
    Q3_REQUIRE(c->layers > 0 && c->pages > 0 && c->kv_heads > 0 && c->max_seqs > 0 && c->max_seq_pages > 0, "pages: non-positive size");
    Q3_REQUIRE(c->layers <= 4096 && c->kv_heads <= 4096 && c->pages <= (1 << 28) && c->max_seqs <= (1 << 24), "pages: size out of range");
    Q3_REQUIRE((int64_t)c->max_seq_pages * c->page_tokens < (1ll << 31), "pages: a sequence may hold fewer than 2^31 tokens");
    Q3_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->table, 4) && aligned(c->lens, 4) && aligned(c->refs, 4) && aligned(c->status, 4),
               "pages: misaligned pointer");
    if (workspace)
        Q3_REQUIRE(c->workspace && aligned(c->workspace, 16) && c->workspace_bytes >= pages_workspace(*c), "pages: workspace missing, misaligned or too small");
}
void check_list(const q3asr_kv_pages* c, int n) { Q3_REQUIRE(n >= 0 && n <= c->max_seqs, "pages: more entries than sequences"); }

void check_batch(const q3asr_kv_pages* c, const q3asr_attn_batch* b) {
    Q3_REQUIRE(b && b->n >= 0 && b->rows >= 0, "pages: bad batch");
    if (b->n == 0 || b->rows == 0) return;
    Q3_REQUIRE(b->seqs && b->cu_rows, "pages: null argument in the batch");
    Q3_REQUIRE(aligned(b->seqs, 4) && aligned(b->cu_rows, 4) && aligned(b->cu_groups, 4) && aligned(b->shared, 4), "pages: misaligned list in the batch");
    Q3_REQUIRE(b->n <= c->max_seqs, "pages: more entries than sequences");
    Q3_REQUIRE(b->rows <= MAX_ROWS, "pages: 2^24 rows or more");
}

// After a call on the model's own stream: errors that the device found become this call's.
void finish(Call& call, const q3asr_kv_pages& c) {
    if (!call.wait) return;
    int32_t st[4];
    HIP_CHECK(hipMemcpyAsync(st, c.status, sizeof st, hipMemcpyDeviceToHost, call.s));
    HIP_CHECK(hipStreamSynchronize(call.s));
    if (st[0] == Q3ASR_PAGES_OK) return;
    launch_pages_clear_status(c, call.s);
    HIP_CHECK(hipStreamSynchronize(call.s));
    const std::string entry = " (entry " + std::to_string(st[1]) + ")";
    switch (st[0]) {
        case Q3ASR_PAGES_BAD_INDEX: throw Q3Error("q3asr: pages: a number out of range" + entry);
        case Q3ASR_PAGES_DUPLICATE: throw Q3Error("q3asr: pages: a sequence is named twice" + entry);
        case Q3ASR_PAGES_NO_PAGES: throw Q3Error("q3asr: pages: not enough free pages (" + std::to_string(st[2]) + " short)");
        case Q3ASR_PAGES_TOO_LONG: throw Q3Error("q3asr: pages: a sequence would outgrow its page table" + entry);
        default: throw Q3Error("q3asr: pages: the batch breaks its bounds, or a page to be written is shared" + entry);
    }
}

}  // namespace

extern "C" {

int q3asr_i8_quantize(q3asr_model* m, const void* x, int dtype, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq,
                      float* scales, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m && x && q && scales, "i8_quantize: null argument");
    Q3_REQUIRE(rows > 0 && cols > 0, "i8_quantize: empty problem");
    Q3_REQUIRE(rows <= MAX_ROWS && cols <= MAX_LD_I8, "i8_quantize: 2^24 rows or more, or more than 4194304 columns");
    check_rows("i8_quantize: x", x, dtype, ldx, cols);
    Q3_REQUIRE(aligned(scales, 4), "i8_quantize: misaligned scales");
    Q3_REQUIRE(aligned(q, 16) && ldq % 16 == 0 && ldq >= (((int64_t)cols + 15) & ~15ll) && ldq < MAX_LD,
               "i8_quantize: rows of q must be aligned to 16 bytes and hold cols rounded up to 16");
    Call call(m, stream);
    launch_i8_quantize({x, dtype == Q3ASR_F32, ldx}, rows, cols, q, ldq, scales, call.s);
    call.done();
    Q3_API_END
}

static void check_product(const int8_t* w, int64_t ldw, const float* w_scales, const float* bias, int M, int N, int K, const void* out, int out_dtype, int64_t ldo) {
    Q3_REQUIRE(w && w_scales && out, "i8: null argument");
    Q3_REQUIRE(M > 0 && N > 0 && K > 0, "i8: empty problem");
    Q3_REQUIRE(K <= I8_MAX_K, "i8: K above 131056 could overflow the 32-bit sums");
    Q3_REQUIRE((int64_t)cdiv(M, 64) * cdiv(N, 64) < (1ll << 31), "i8: too many output tiles");
    Q3_REQUIRE(M <= MAX_ROWS && N <= MAX_ROWS, "i8: 2^24 rows or output channels, or more");
    check_i8("i8: w", w, ldw, K);
    check_rows("i8: out", out, out_dtype, ldo, N);
    Q3_REQUIRE(aligned(w_scales, 4) && aligned(bias, 4), "i8: misaligned scales or bias");
}

int q3asr_i8_matmul(q3asr_model* m, const int8_t* a, int64_t lda, const float* a_scales, const int8_t* w, int64_t ldw,
                    const float* w_scales, const float* bias, int M, int N, int K, void* out, int out_dtype, int64_t ldo, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m && a && a_scales, "i8_matmul: null argument");
    check_product(w, ldw, w_scales, bias, M, N, K, out, out_dtype, ldo);
    Q3_REQUIRE(K % 16 == 0, "i8_matmul: K must be a multiple of 16");
    check_i8("i8: a", a, lda, K);
    Q3_REQUIRE(aligned(a_scales, 4), "i8_matmul: misaligned scales");
    Call call(m, stream);
    I8Params p;
    p.A = a; p.lda = lda; p.sa = a_scales; p.W = w; p.ldw = ldw; p.sw = w_scales; p.bias = bias;
    p.M = M; p.N = N; p.K = K; p.out = out; p.ldo = ldo; p.out_f32 = out_dtype == Q3ASR_F32;
    launch_i8_matmul(p, call.s);
    call.done();
    Q3_API_END
}

int q3asr_i8_linear(q3asr_model* m, const void* x, int x_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scales,
                    const float* bias, int M, int N, int K, void* out, int out_dtype, int64_t ldo, void* workspace,
                    int64_t workspace_bytes, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m && x && workspace, "i8_linear: null argument");
    check_product(w, ldw, w_scales, bias, M, N, K, out, out_dtype, ldo);
    check_rows("i8_linear: x", x, x_dtype, ldx, K);
    Q3_REQUIRE(aligned(workspace, 16), "i8_linear: misaligned workspace");
    Q3_REQUIRE(workspace_bytes >= quantized_bytes(M, K), "i8_linear: workspace too small");
    Call call(m, stream);
    I8Params p;
    p.A = (const int8_t*)workspace; p.lda = (K + 15) & ~15;
    p.sa = (const float*)((char*)workspace + round256((int64_t)M * p.lda));
    p.W = w; p.ldw = ldw; p.sw = w_scales; p.bias = bias;
    p.M = M; p.N = N; p.K = K; p.out = out; p.ldo = ldo; p.out_f32 = out_dtype == Q3ASR_F32;
    const I8Source src{x, x_dtype == Q3ASR_F32, ldx};
    if (!launch_i8_linear_few_rows(p, src, call.s)) {
        launch_i8_quantize(src, M, K, (int8_t*)p.A, p.lda, (float*)p.sa, call.s);
        launch_i8_matmul(p, call.s);
    }
    call.done();
    Q3_API_END
}

int64_t q3asr_i8_workspace(q3asr_model* m, int M, int N, int K) {
    if (!m || M <= 0 || N <= 0 || K <= 0 || K > I8_MAX_K || M > MAX_ROWS || N > MAX_ROWS) return -1;
    return quantized_bytes(M, K);
}

int q3asr_pages_status(q3asr_model* m, const q3asr_kv_pages* c, int32_t* out, int clear, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m && out, "pages_status: null argument");
    check_cache(c, false);
    Call call(m, stream);
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    HIP_CHECK(hipStreamIsCapturing(call.s, &cap));
    Q3_REQUIRE(cap == hipStreamCaptureStatusNone, "pages_status: not under graph capture");
    HIP_CHECK(hipMemcpyAsync(out, c->status, 16, hipMemcpyDeviceToHost, call.s));
    HIP_CHECK(hipStreamSynchronize(call.s));
    if (clear) {
        launch_pages_clear_status(*c, call.s);
        HIP_CHECK(hipStreamSynchronize(call.s));
    }
    Q3_API_END
}

int64_t q3asr_pages_workspace(const q3asr_kv_pages* c) {
    return c && c->pages > 0 && c->max_seqs > 0 && c->max_seq_pages > 0 ? pages_workspace(*c) : -1;
}

int q3asr_pages_reset(q3asr_model* m, const q3asr_kv_pages* c, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_reset: null model");
    check_cache(c, false);
    Call call(m, stream);
    launch_pages_reset(*c, call.s);
    finish(call, *c);
    Q3_API_END
}

int q3asr_pages_fork(q3asr_model* m, const q3asr_kv_pages* c, const int32_t* dst, const int32_t* src, int n, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_fork: null model");
    check_cache(c, true);
    check_list(c, n);
    Q3_REQUIRE(n == 0 || (dst && src), "pages_fork: null argument");
    Q3_REQUIRE(aligned(dst, 4) && aligned(src, 4), "pages_fork: misaligned list");
    Call call(m, stream);
    if (n > 0) launch_pages_fork(*c, dst, src, n, call.s);
    finish(call, *c);
    Q3_API_END
}

int q3asr_pages_free(q3asr_model* m, const q3asr_kv_pages* c, const int32_t* seqs, int n, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_free: null model");
    check_cache(c, true);
    check_list(c, n);
    Q3_REQUIRE(n == 0 || seqs, "pages_free: null argument");
    Q3_REQUIRE(aligned(seqs, 4), "pages_free: misaligned list");
    Call call(m, stream);
    if (n > 0) launch_pages_fork(*c, seqs, nullptr, n, call.s);
    finish(call, *c);
    Q3_API_END
}

int q3asr_pages_reserve(q3asr_model* m, const q3asr_kv_pages* c, const int32_t* seqs, const int32_t* tokens, int n, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_reserve: null model");
    check_cache(c, true);
    check_list(c, n);
    Q3_REQUIRE(n == 0 || (seqs && tokens), "pages_reserve: null argument");
    Q3_REQUIRE(aligned(seqs, 4) && aligned(tokens, 4), "pages_reserve: misaligned list");
    Call call(m, stream);
    if (n > 0) launch_pages_reserve(*c, seqs, tokens, n, call.s);
    finish(call, *c);
    Q3_API_END
}

int q3asr_pages_compact(q3asr_model* m, const q3asr_kv_pages* c, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_compact: null model");
    check_cache(c, true);
    Call call(m, stream);
    launch_pages_compact(*c, call.s);
    finish(call, *c);
    Q3_API_END
}

int q3asr_pages_write(q3asr_model* m, const q3asr_kv_pages* c, int layer, const uint16_t* k_rows, int64_t k_ld,
                      const uint16_t* v_rows, int64_t v_ld, const q3asr_attn_batch* b, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "pages_write: null model");
    check_cache(c, false);
    check_batch(c, b);
    Q3_REQUIRE(layer >= 0 && layer < c->layers, "pages_write: layer out of range");
    const bool any = b->n > 0 && b->rows > 0;
    if (any) {
        Q3_REQUIRE(k_rows && v_rows, "pages_write: null argument");
        const int64_t width = (int64_t)c->kv_heads * c->head_dim;
        Q3_REQUIRE(k_ld >= width && v_ld >= width && k_ld % 8 == 0 && v_ld % 8 == 0 && k_ld < MAX_LD && v_ld < MAX_LD && aligned(k_rows, 16) &&
                       aligned(v_rows, 16),
                   "pages_write: rows must hold all KV heads and be aligned to 16 bytes");
    }
    Call call(m, stream);
    if (any) launch_pages_write(*c, layer, k_rows, k_ld, v_rows, v_ld, *b, call.s);
    finish(call, *c);
    Q3_API_END
}

static void check_attention(const q3asr_kv_pages* c, const q3asr_attn_batch* b, int heads) {
    check_batch(c, b);
    Q3_REQUIRE(heads > 0 && heads % c->kv_heads == 0 && heads <= (1 << 16), "paged_attention: heads must be a multiple of the KV heads");
    if (b->n == 0 || b->rows == 0) return;
    Q3_REQUIRE((int64_t)b->rows * heads < (1ll << 31), "paged_attention: too many rows");
    Q3_REQUIRE(b->max_rows >= 1 && b->max_rows <= b->rows, "paged_attention: max_rows must lie between 1 and rows");
    Q3_REQUIRE(b->max_len >= 0 && b->max_len <= (int64_t)c->max_seq_pages * c->page_tokens, "paged_attention: max_len beyond a page table");
    Q3_REQUIRE(b->n_groups >= 0 && b->n_groups <= b->n, "paged_attention: more groups than sequences");
    if (b->n_groups > 0) {
        Q3_REQUIRE(b->cu_groups && b->shared, "paged_attention: groups without their arrays");
        Q3_REQUIRE(b->max_group_rows >= b->max_rows && b->max_group_rows <= b->rows, "paged_attention: max_group_rows must lie between max_rows and rows");
        Q3_REQUIRE(b->max_shared >= 0 && b->max_shared <= b->max_len && b->max_own >= 0 && b->max_own <= b->max_len,
                   "paged_attention: max_shared and max_own must lie between 0 and max_len");
    }
    // tiles of 32 keys by 16 rows, and one for every beginning, are counted in 32 bits: at most one incomplete tile of rows per sequence
    // and group and KV head, twice for shared and own keys
    const int64_t tiles = ((int64_t)b->max_len + 63) / 32, streams = ((int64_t)b->rows * heads + 15) / 16 + (int64_t)b->n * c->kv_heads;
    Q3_REQUIRE(2 * streams < ((1ll << 31) - (1 << 16)) / tiles, "paged_attention: too many rows for so many tokens in one call");
}

int64_t q3asr_paged_attention_workspace(q3asr_model* m, const q3asr_kv_pages* c, const q3asr_attn_batch* b, int heads) {
    if (!m) return -1;
    try {
        check_cache(c, false);
        check_attention(c, b, heads);
        if (b->n == 0 || b->rows == 0) return 0;
        return paged_attention_workspace(*c, *b, heads);
    } catch (const std::exception& e) {
        q3_set_error(e.what());
    } catch (...) {
        q3_set_error("q3asr: unknown error");
    }
    return -1;
}

int q3asr_paged_attention(q3asr_model* m, const q3asr_kv_pages* c, int layer, const uint16_t* q, int64_t q_ld, int heads,
                          float scale, const q3asr_attn_batch* b, uint16_t* out, int64_t o_ld, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream) {
    Q3_API_BEGIN
    Q3_REQUIRE(m, "paged_attention: null model");
    check_cache(c, false);
    check_attention(c, b, heads);
    Q3_REQUIRE(layer >= 0 && layer < c->layers, "paged_attention: layer out of range");
    const bool any = b->n > 0 && b->rows > 0;
    if (any) {
        Q3_REQUIRE(q && out, "paged_attention: null argument");
        const int64_t width = (int64_t)heads * c->head_dim;
        Q3_REQUIRE(q_ld >= width && o_ld >= width && q_ld % 8 == 0 && o_ld % 8 == 0 && q_ld < MAX_LD && o_ld < MAX_LD && aligned(q, 16) &&
                       aligned(out, 16) && aligned(lse, 4),
                   "paged_attention: rows of q and out must hold all heads and be aligned to 16 bytes");
        Q3_REQUIRE(scale > -1e30f && scale < 1e30f, "paged_attention: scale must be finite and below 1e30");
        const int64_t need = paged_attention_workspace(*c, *b, heads);
        Q3_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), "paged_attention: workspace missing, misaligned or too small");
    }
    Call call(m, stream);
    if (any) launch_paged_attention(*c, layer, q, q_ld, heads, scale, *b, out, o_ld, lse, workspace, call.s);
    finish(call, *c);
    Q3_API_END
}

}  // extern "C"
