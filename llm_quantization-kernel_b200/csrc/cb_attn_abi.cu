// extern "C" entry points of the attention operators: argument checks and kernel choice.
#include <cmath>

#include "cb_common.cuh"
#include "cb_kv4.cuh"

namespace cb {

int launch_kv4_rows(bool append, const cb_kv4_cache* c, const void* k_in, const void* v_in, const int64_t* strides, void* k_out,
                    void* v_out, int64_t n_tokens, const int32_t* table, int64_t table_stride, int64_t n_seqs,
                    const int32_t* starts, const int32_t* cu, cudaStream_t stream);
int launch_kv4_attention(const cb_kv4_cache* c, const void* q, const int64_t* q_strides, void* out, int64_t B, int64_t T, int64_t H,
                         const int32_t* table, int64_t table_stride, const int32_t* lengths, float scale, int* counters,
                         float* partial, cudaStream_t stream);
int64_t kv4_attention_segments(int64_t B, int64_t rows, int64_t kv_heads);
size_t kv4_attention_partial_bytes(int64_t rows, int head_dim);

int launch_prompt_attention(const void* q, const void* k, const void* v, const int64_t* strides, void* out, int64_t Tq, int64_t Tk,
                            int64_t H, int64_t Hkv, int head_dim, int dtype, const int32_t* cu_q, const int32_t* cu_k, int64_t B,
                            float scale, int causal, int* counters, float* partial, cudaStream_t stream);
int64_t prompt_attention_parts(int64_t Tq, int64_t Tk, int64_t H, int64_t B);
int64_t prompt_attention_most_parts();
size_t prompt_attention_partial_bytes(int64_t parts, int head_dim);
size_t prompt_attention_counter_bytes(int64_t parts);

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Does `out` (bytes) meet the stretch from the first to the last byte of the 16-bit values at p[i0 * s0 + i1 * s1 + i2 * s2 + d]?  A CTA writes rows of the
// output while others still read the queries, keys and values of theirs.
bool meets(const void* out, int64_t bytes, const void* p, int head_dim, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2 = 1, int64_t s2 = 0) {
    if (p == nullptr || n0 <= 0 || n1 <= 0 || n2 <= 0) return false;
    const int64_t ends[3] = {(n0 - 1) * s0, (n1 - 1) * s1, (n2 - 1) * s2};
    intptr_t lo = reinterpret_cast<intptr_t>(p), hi = lo + 2ll * head_dim;
    for (int64_t e : ends) (e < 0 ? lo : hi) += 2 * e;
    const intptr_t o = reinterpret_cast<intptr_t>(out);
    return o < hi && lo < o + bytes;
}

int64_t block_bytes(int head_dim, int group_size) {
    if ((head_dim != 64 && head_dim != 128) || (group_size != 32 && group_size != 64 && group_size != 128) || group_size > head_dim) return 0;
    return 2 * kKvBlock * (head_dim / 2 + 4 * (head_dim / group_size));
}

int check_cache(const char* who, const cb_kv4_cache* c) {
    CB_REQUIRE(c != nullptr, "%s: cache record is NULL", who);
    CB_REQUIRE(c->dtype == CB_F16 || c->dtype == CB_BF16, "%s: the cache's dtype must be fp16 or bf16", who);
    CB_REQUIRE(block_bytes(c->head_dim, c->group_size) != 0,
               "%s: head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim (got %d, %d)", who, c->head_dim, c->group_size);
    CB_REQUIRE(c->page_size >= kKvBlock && c->page_size % kKvBlock == 0 && c->page_size <= (1 << 20),
               "%s: page_size must be a multiple of 16", who);
    CB_REQUIRE(c->kv_heads > 0 && c->kv_heads < (1 << 16), "%s: kv_heads out of range", who);
    CB_REQUIRE(c->n_pages >= 0 && c->n_pages < (1ll << 31), "%s: n_pages out of range", who);
    CB_REQUIRE(c->pages != nullptr && aligned16(c->pages), "%s: pages must be a 16-byte aligned pointer", who);
    return CB_OK;
}

int check_rows(const char* who, const cb_kv4_cache* c, const void* k, const void* v, int64_t n_tokens, const int32_t* table,
               int64_t table_stride, int64_t n_seqs, const int32_t* starts, const int32_t* cu) {
    const int rc = check_cache(who, c);
    if (rc != CB_OK) return rc;
    CB_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 31), "%s: n_tokens out of range", who);
    CB_REQUIRE(n_seqs >= 0 && n_seqs < (1ll << 31) && table_stride >= 0 && table_stride < (1ll << 31), "%s: page table out of range", who);
    if (n_tokens == 0) return CB_OK;
    CB_REQUIRE(n_seqs > 0, "%s: tokens without a sequence", who);
    CB_REQUIRE(cu != nullptr || n_tokens % n_seqs == 0, "%s: without cu_seqlens every sequence has as many tokens", who);
    CB_REQUIRE(k && v && starts && (table || table_stride == 0), "%s: NULL pointer", who);
    CB_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", who);
    return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" {

size_t cb_kv4_block_bytes(int head_dim, int group_size) { return (size_t)block_bytes(head_dim, group_size); }

int cb_kv4_append(const cb_kv4_cache* cache, const void* k, const void* v, const int64_t* strides4, int64_t n_tokens,
                  const int32_t* page_table, int64_t table_stride, int64_t n_seqs, const int32_t* starts,
                  const int32_t* cu_seqlens, void* stream) {
    const int rc = check_rows("kv4_append", cache, k, v, n_tokens, page_table, table_stride, n_seqs, starts, cu_seqlens);
    if (rc != CB_OK || n_tokens == 0) return rc;
    CB_REQUIRE(strides4 != nullptr, "kv4_append: strides are NULL");
    for (int i = 0; i < 4; ++i) CB_REQUIRE(strides4[i] % 8 == 0, "kv4_append: strides must be multiples of 8 elements");
    return launch_kv4_rows(true, cache, k, v, strides4, nullptr, nullptr, n_tokens, page_table, table_stride, n_seqs, starts,
                           cu_seqlens, reinterpret_cast<cudaStream_t>(stream));
}

int cb_kv4_read(const cb_kv4_cache* cache, void* k, void* v, int64_t n_tokens, const int32_t* page_table, int64_t table_stride,
                int64_t n_seqs, const int32_t* starts, const int32_t* cu_seqlens, void* stream) {
    const int rc = check_rows("kv4_read", cache, k, v, n_tokens, page_table, table_stride, n_seqs, starts, cu_seqlens);
    if (rc != CB_OK || n_tokens == 0) return rc;
    return launch_kv4_rows(false, cache, nullptr, nullptr, nullptr, k, v, n_tokens, page_table, table_stride, n_seqs, starts,
                           cu_seqlens, reinterpret_cast<cudaStream_t>(stream));
}

int64_t cb_kv4_attention_counters(int64_t B, int64_t T, int64_t H, int64_t kv_heads) {
    if (B <= 0 || T <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads != 0) return 0;
    return kv4_attention_segments(B, T * (H / kv_heads), kv_heads);
}

size_t cb_kv4_attention_partial_bytes(int64_t T, int64_t H, int64_t kv_heads, int head_dim) {
    if (T <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads != 0) return 0;
    return kv4_attention_partial_bytes(T * (H / kv_heads), head_dim);
}

int cb_kv4_attention(const cb_kv4_cache* cache, const void* q, const int64_t* strides3, void* out, int64_t B, int64_t T, int64_t H,
                     const int32_t* page_table, int64_t table_stride, const int32_t* lengths, float scale, void* counters,
                     size_t counter_bytes, void* partial, size_t partial_bytes, void* stream) {
    const char* who = "kv4_attention";
    const int rc = check_cache(who, cache);
    if (rc != CB_OK) return rc;
    CB_REQUIRE(B >= 0 && B < (1ll << 31) && T >= 0 && H >= 0, "%s: negative or too large batch, T or H", who);
    CB_REQUIRE(table_stride >= 0 && table_stride < (1ll << 31), "%s: page table out of range", who);
    CB_REQUIRE(std::isfinite(scale), "%s: scale must be finite", who);
    if (B == 0 || T == 0 || H == 0) return CB_OK;
    CB_REQUIRE(H % cache->kv_heads == 0, "%s: H must be a multiple of kv_heads", who);
    CB_REQUIRE(T < (1 << 24) && H < (1 << 20) && T * H * cache->head_dim < (1ll << 31), "%s: T * H out of range", who);
    const int64_t segs = cb_kv4_attention_counters(B, T, H, cache->kv_heads);
    // the kernel numbers blocks, and a few more for each segment, with 32 bits
    CB_REQUIRE(segs < (1ll << 26) && (table_stride * (cache->page_size / kKvBlock) + 256) < (1ll << 31) / segs,
               "%s: too many rows and pages", who);
    CB_REQUIRE(q && out && lengths && strides3 && (page_table || table_stride == 0), "%s: NULL pointer", who);
    CB_REQUIRE(aligned16(q) && aligned16(out), "%s: q and out must be 16-byte aligned", who);
    for (int i = 0; i < 3; ++i) CB_REQUIRE(strides3[i] % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    CB_REQUIRE(counters != nullptr && counter_bytes >= (size_t)segs * sizeof(int), "%s: needs %lld zeroed counters", who, (long long)segs);
    const size_t need = cb_kv4_attention_partial_bytes(T, H, cache->kv_heads, cache->head_dim);
    CB_REQUIRE(partial != nullptr && partial_bytes >= need && aligned16(partial), "%s: needs %zu bytes of 16-byte aligned scratch", who, need);
    CB_REQUIRE(!meets(out, 2 * B * T * H * cache->head_dim, q, cache->head_dim, B, strides3[0], T, strides3[1], H, strides3[2]),
               "%s: out and q share memory", who);
    return launch_kv4_attention(cache, q, strides3, out, B, T, H, page_table, table_stride, lengths, scale,
                                reinterpret_cast<int*>(counters), reinterpret_cast<float*>(partial),
                                reinterpret_cast<cudaStream_t>(stream));
}

size_t cb_prompt_attention_scratch(int head_dim, size_t* counter_bytes) {
    const int64_t parts = prompt_attention_most_parts();
    if (counter_bytes != nullptr) *counter_bytes = prompt_attention_counter_bytes(parts);
    return prompt_attention_partial_bytes(parts, head_dim);
}

size_t cb_prompt_attention_scratch_for(int64_t Tq, int64_t Tk, int64_t H, int64_t B, int head_dim, size_t* counter_bytes) {
    const int64_t parts = Tq <= 0 || Tk <= 0 || H <= 0 || B <= 0 ? 0 : prompt_attention_parts(Tq, Tk, H, B);
    if (counter_bytes != nullptr) *counter_bytes = prompt_attention_counter_bytes(parts);
    return prompt_attention_partial_bytes(parts, head_dim);
}

int cb_prompt_attention(const void* q, const void* k, const void* v, const int64_t* strides6, void* out, int64_t Tq, int64_t Tk,
                        int64_t H, int64_t Hkv, int head_dim, int dtype, const int32_t* cu_q, const int32_t* cu_k, int64_t B,
                        float scale, int causal, void* counters, size_t counter_bytes, void* partial, size_t partial_bytes,
                        void* stream) {
    const char* who = "prompt_attention";
    CB_REQUIRE(dtype == CB_F16 || dtype == CB_BF16, "%s: dtype must be fp16 or bf16", who);
    CB_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128 (got %d)", who, head_dim);
    CB_REQUIRE(Tq >= 0 && Tk >= 0 && Tq < (1ll << 30) && Tk < (1ll << 30), "%s: too many tokens", who);
    CB_REQUIRE(H >= 0 && Hkv >= 0 && H < (1 << 20) && Hkv < (1 << 20) && B >= 0, "%s: heads or sequences out of range", who);
    // every CTA walks over the bounds of all sequences, a microsecond for 32 of them, while its other warps wait with a limit of a second
    CB_REQUIRE(B <= (1ll << 22), "%s: more than 2^22 sequences", who);
    CB_REQUIRE(std::isfinite(scale), "%s: scale must be finite", who);
    if (Tq == 0 || H == 0 || B == 0) return CB_OK;
    CB_REQUIRE(Hkv > 0 && H % Hkv == 0, "%s: H must be a multiple of Hkv", who);
    CB_REQUIRE(q && out && cu_q && cu_k && strides6 && (Tk == 0 || (k && v)), "%s: NULL pointer", who);
    CB_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "%s: q, k, v and out must be 16-byte aligned", who);
    for (int i = 0; i < 6; ++i) {
        const int64_t used = i == 0 ? Tq : i == 1 ? H : (i & 1) ? Hkv : Tk;
        CB_REQUIRE(used <= 1 || (strides6[i] > 0 && strides6[i] % 8 == 0 && strides6[i] < (1ll << 38)),
                   "%s: strides must be positive multiples of 8 elements", who);
    }
    const int64_t parts = prompt_attention_parts(Tq, Tk, H, B);
    CB_REQUIRE(counters != nullptr && counter_bytes >= prompt_attention_counter_bytes(parts) && partial != nullptr && aligned16(partial) &&
                   partial_bytes >= prompt_attention_partial_bytes(parts, head_dim),
               "%s: scratch is missing or too small (cb_prompt_attention_scratch)", who);
    const int64_t out_bytes = 2 * Tq * H * head_dim;
    CB_REQUIRE(!meets(out, out_bytes, q, head_dim, Tq, strides6[0], H, strides6[1]) && !meets(out, out_bytes, k, head_dim, Tk, strides6[2], Hkv, strides6[3]) &&
                   !meets(out, out_bytes, v, head_dim, Tk, strides6[4], Hkv, strides6[5]), "%s: out shares memory with q, k or v", who);
    return launch_prompt_attention(q, k, v, strides6, out, Tq, Tk, H, Hkv, head_dim, dtype, cu_q, cu_k, B, scale, causal,
                                   reinterpret_cast<int*>(counters), reinterpret_cast<float*>(partial), reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
