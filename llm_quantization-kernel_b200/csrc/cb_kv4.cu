// Writing to and reading from the 4-bit key/value cache (layout: cb_kv4.cuh).
//
//   lo = min(x), scale = round_T((max(x) - lo) / 15), code = round_half_even((x - lo) / scale) <= 15, value = code * scale + lo
//
// over the GS values x of a group, T the cache's 16-bit type.  A group with an infinity or a NaN keeps NaN for both and
// reads back as NaN; a scale below the smallest normal float is kept as 0, and the group reads back as lo.
//
// Both kernels are bound by memory: 2 bytes of a value on one side, 0.5 + 4 / GS on the other.  A thread owns 8
// consecutive values of one row (token, head, K or V): one 16-byte access on the 16-bit side, one 4-byte word of codes on
// the other.  A CTA takes 16 tokens and a few heads, the tokens along its threads, so that what it writes is contiguous
// on both sides; it looks its 16 tokens' pages up once.
#include <algorithm>

#include "cb_kv4.cuh"

namespace cb {
namespace {

constexpr int kTok = 16;              // tokens of a CTA
constexpr int kThreads = 256;
__device__ int g_kv4_status;

struct RowParams {
    Kv4View c;
    const int32_t* starts;            // [n_seqs] position of each sequence's first token
    const int32_t* cu;                // [n_seqs + 1] first token of each sequence, or nullptr: per_seq tokens each
    int64_t n_tokens, n_seqs, per_seq;
    const void* k_in; const void* v_in;       // append
    int64_t k_tok, k_head, v_tok, v_head;     // their strides in elements
    void* k_out; void* v_out;                 // read: [n_tokens, kv_heads, D]
    int heads_per_cta;
};

// Page and position inside it of packed token `tok`; page -1: no such place.
__device__ __forceinline__ void find_slot(const RowParams& P, int64_t tok, int& page, int& off) {
    page = -1; off = 0;
    if (tok >= P.n_tokens) return;
    int64_t b, first;
    if (P.cu != nullptr) {
        int64_t lo = 0, hi = P.n_seqs;            // the last sequence that begins at or before tok
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (P.cu[mid] <= tok) lo = mid; else hi = mid;
        }
        b = lo;
        first = P.cu[b];
        if (tok < first || tok >= P.cu[b + 1]) return;
    } else {
        b = tok / P.per_seq;
        first = b * P.per_seq;
    }
    const int64_t pos = (int64_t)P.starts[b] + (tok - first), ps = (int64_t)P.c.blocks_per_page * kKvBlock;
    if (pos < 0 || pos >= P.c.table_stride * ps) { atomicExch(&g_kv4_status, kKv4BadPage); return; }
    const int64_t pg = P.c.table[b * P.c.table_stride + pos / ps];
    if (pg < 0 || pg >= P.c.n_pages) { atomicExch(&g_kv4_status, kKv4BadPage); return; }
    page = (int)pg;
    off = (int)(pos % ps);
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    using V2 = __half2;
    __device__ static float2 f2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    __device__ static uint32_t min2(uint32_t a, uint32_t b) {
        const __half2 r = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ static uint32_t max2(uint32_t a, uint32_t b) {
        const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ static uint32_t pack(float a, float b) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
template <> struct Pair<__nv_bfloat16> {
    using V2 = __nv_bfloat162;
    __device__ static float2 f2(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    __device__ static uint32_t min2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ static uint32_t max2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ static uint32_t pack(float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

// The group's (scale, lo) as stored, from its exact minimum and maximum.
template <typename T>
__device__ __forceinline__ uint32_t group_meta(float lo, float hi) {
    float scale = to_f32(from_f32<T>(__fdiv_rn(hi - lo, 15.0f)));
    if (scale < 1.17549435e-38f) scale = 0.f;
    if (!(scale < INFINITY) || !(fabsf(lo) < INFINITY)) scale = lo = __int_as_float(0x7fffffff);
    return Pair<T>::pack(scale, lo);
}

// round_half_even((x - lo) / scale), at most 15.  x * inv may miss a tie or fall on the wrong side of one; the remainder
// c * scale - (x - lo), which the fused multiply-add forms without rounding, puts that right.
__device__ __forceinline__ uint32_t code_of(float x, float lo, float scale, float inv) {
    const float a = x - lo, h = 0.5f * scale;
    float c = rintf(a * inv);
    const float d = fmaf(-c, scale, a);
    const bool odd = ((int)c & 1) != 0;
    if (d > h || (d == h && odd)) c += 1.f;
    if (d < -h || (d == -h && odd)) c -= 1.f;
    return (uint32_t)(int)fminf(c, 15.f);
}

template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads)
kv4_append_kernel(const RowParams P) {
    using L = KvLayout<D, GS>;
    constexpr int kTpr = D / 8;                        // threads of a row
    constexpr int kPer = kThreads / (kTpr * kTok);     // rows of each token side by side: 1 at D = 128, 2 at 64
    constexpr int kBatch = 4;                          // loads in flight
    __shared__ int s_page[kTok], s_off[kTok];
    const int tid = threadIdx.x;
    if (tid < kTok) find_slot(P, (int64_t)blockIdx.x * kTok + tid, s_page[tid], s_off[tid]);
    const int part = tid % kTpr, tok = (tid / kTpr) % kTok, sub = tid / (kTpr * kTok);
    const int h0 = blockIdx.y * P.heads_per_cta, h1 = min(h0 + P.heads_per_cta, P.c.kv_heads);
    const int64_t token = (int64_t)blockIdx.x * kTok + tok;
    const int rows = 2 * (h1 - h0);                    // (head, K or V)
    __syncthreads();
    const int page = s_page[tok], off = s_off[tok], in_block = off % kKvBlock;
    const bool live = page >= 0;
    for (int r0 = sub; r0 < rows; r0 += kPer * kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kPer;
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (live && r < rows) {
                const int h = h0 + (r >> 1);
                const T* src = (r & 1) ? reinterpret_cast<const T*>(P.v_in) + token * P.v_tok + h * P.v_head
                                       : reinterpret_cast<const T*>(P.k_in) + token * P.k_tok + h * P.k_head;
                x[i] = __ldg(reinterpret_cast<const uint4*>(src + part * 8));
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kPer;
            // all lanes take part in the shuffles; what dead ones compute is dropped
            uint32_t mn = Pair<T>::min2(Pair<T>::min2(x[i].x, x[i].y), Pair<T>::min2(x[i].z, x[i].w));
            uint32_t mx = Pair<T>::max2(Pair<T>::max2(x[i].x, x[i].y), Pair<T>::max2(x[i].z, x[i].w));
            mn = Pair<T>::min2(mn, __byte_perm(mn, 0u, 0x1032));
            mx = Pair<T>::max2(mx, __byte_perm(mx, 0u, 0x1032)) ^ 0x80008000u;
            uint32_t both = __byte_perm(mn, mx, 0x5410);                  // (min, -max)
#pragma unroll
            for (int o = 1; o < GS / 8; o <<= 1) both = Pair<T>::min2(both, __shfl_xor_sync(0xffffffffu, both, o));
            const float2 mm = Pair<T>::f2(both);
            const uint32_t meta = group_meta<T>(mm.x, -mm.y);
            const float2 sl = Pair<T>::f2(meta);
            const float inv = sl.x > 0.f ? __frcp_rn(sl.x) : 0.f;
            uint32_t word = 0u;
            const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            if (sl.x > 0.f) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = Pair<T>::f2(xs[j]);
                    word |= code_of(f.x, sl.y, sl.x, inv) << (8 * j);
                    word |= code_of(f.y, sl.y, sl.x, inv) << (8 * j + 4);
                }
            }
            if (live && r < rows) {
                const int h = h0 + (r >> 1);
                unsigned char* blk = P.c.pages + (((int64_t)page * P.c.kv_heads + h) * P.c.blocks_per_page + off / kKvBlock) * L::kBytes;
                const int d = part * 8;
                const bool lead = d % GS == 0;
                if ((r & 1) == 0) {
                    *reinterpret_cast<uint32_t*>(blk + in_block * L::kRow + L::k_nibble(d) / 2) = word;
                    if (lead) *reinterpret_cast<uint32_t*>(blk + L::kKMeta + in_block * L::kMeta + (d / GS) * 4) = meta;
                } else {
                    *reinterpret_cast<uint16_t*>(blk + L::kVCodes + L::v_byte(d, in_block)) = (uint16_t)word;
                    *reinterpret_cast<uint16_t*>(blk + L::kVCodes + L::v_byte(d + 4, in_block)) = (uint16_t)(word >> 16);
                    if (lead) *reinterpret_cast<uint32_t*>(blk + L::kVMeta + in_block * L::kMeta + (d / GS) * 4) = meta;
                }
            }
        }
    }
}

// code * scale + lo, at most the type's largest number in size: the rounding of scale can carry the largest value of a
// group whose range reaches that number past it.  NaN stays.
template <typename T>
__device__ __forceinline__ float value_of(float code, float scale, float lo) {
    const float v = fmaf(code, scale, lo), top = std::is_same<T, __half>::value ? 65504.f : 3.3895314e38f;
    return v > top ? top : v < -top ? -top : v;
}

template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const RowParams P) {
    using L = KvLayout<D, GS>;
    constexpr int kTpr = D / 8, kPer = kThreads / (kTpr * kTok), kBatch = 4;
    __shared__ int s_page[kTok], s_off[kTok];
    const int tid = threadIdx.x;
    if (tid < kTok) find_slot(P, (int64_t)blockIdx.x * kTok + tid, s_page[tid], s_off[tid]);
    const int part = tid % kTpr, tok = (tid / kTpr) % kTok, sub = tid / (kTpr * kTok);
    const int h0 = blockIdx.y * P.heads_per_cta, h1 = min(h0 + P.heads_per_cta, P.c.kv_heads);
    const int64_t token = (int64_t)blockIdx.x * kTok + tok;
    const int rows = 2 * (h1 - h0), d = part * 8;
    __syncthreads();
    const int page = s_page[tok], off = s_off[tok], in_block = off % kKvBlock;
    if (page < 0) return;
    for (int r0 = sub; r0 < rows; r0 += kPer * kBatch) {
        uint32_t word[kBatch], meta[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kPer;
            word[i] = meta[i] = 0u;
            if (r < rows) {
                const unsigned char* blk = P.c.pages + (((int64_t)page * P.c.kv_heads + h0 + (r >> 1)) * P.c.blocks_per_page + off / kKvBlock) * L::kBytes;
                if ((r & 1) == 0) {
                    word[i] = *reinterpret_cast<const uint32_t*>(blk + in_block * L::kRow + L::k_nibble(d) / 2);
                    meta[i] = *reinterpret_cast<const uint32_t*>(blk + L::kKMeta + in_block * L::kMeta + (d / GS) * 4);
                } else {
                    word[i] = *reinterpret_cast<const uint16_t*>(blk + L::kVCodes + L::v_byte(d, in_block)) |
                              ((uint32_t)*reinterpret_cast<const uint16_t*>(blk + L::kVCodes + L::v_byte(d + 4, in_block)) << 16);
                    meta[i] = *reinterpret_cast<const uint32_t*>(blk + L::kVMeta + in_block * L::kMeta + (d / GS) * 4);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kPer;
            if (r >= rows) continue;
            const float2 sl = Pair<T>::f2(meta[i]);
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // 2^23 + code, exactly, from the bits; a single rounding to fp32, one to T
                const float c0 = __uint_as_float(0x4B000000u | ((word[i] >> (8 * j)) & 15u)) - 8388608.f;
                const float c1 = __uint_as_float(0x4B000000u | ((word[i] >> (8 * j + 4)) & 15u)) - 8388608.f;
                o[j] = Pair<T>::pack(value_of<T>(c0, sl.x, sl.y), value_of<T>(c1, sl.x, sl.y));
            }
            T* dst = ((r & 1) ? reinterpret_cast<T*>(P.v_out) : reinterpret_cast<T*>(P.k_out)) +
                     (token * P.c.kv_heads + h0 + (r >> 1)) * D + d;
            *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

template <typename T, int D, int GS>
int launch_rows_t(bool append, RowParams& P, dim3 grid, cudaStream_t stream) {
    if (append) kv4_append_kernel<T, D, GS><<<grid, kThreads, 0, stream>>>(P);
    else kv4_read_kernel<T, D, GS><<<grid, kThreads, 0, stream>>>(P);
    CB_CUDA_TRY(cudaGetLastError());
    return CB_OK;
}

}  // namespace

// Arguments are checked by the caller.
int launch_kv4_rows(bool append, const cb_kv4_cache* c, const void* k_in, const void* v_in, const int64_t* strides, void* k_out,
                    void* v_out, int64_t n_tokens, const int32_t* table, int64_t table_stride, int64_t n_seqs,
                    const int32_t* starts, const int32_t* cu, cudaStream_t stream) {
    RowParams P{};
    P.c = Kv4View{reinterpret_cast<unsigned char*>(c->pages), c->n_pages, (int)c->kv_heads, c->page_size / kKvBlock, table, table_stride};
    P.starts = starts; P.cu = cu; P.n_tokens = n_tokens; P.n_seqs = n_seqs; P.per_seq = cu == nullptr ? n_tokens / n_seqs : 0;
    P.k_in = k_in; P.v_in = v_in; P.k_out = k_out; P.v_out = v_out;
    if (strides != nullptr) { P.k_tok = strides[0]; P.k_head = strides[1]; P.v_tok = strides[2]; P.v_head = strides[3]; }
    const int sms = sm_count_current();
    if (sms <= 0) return CB_ERR_CUDA;
    // few tokens: one head to a CTA, so that a decode step spreads over the SMs; many: eight, to look pages up less often
    const int64_t tiles = (n_tokens + kTok - 1) / kTok;
    int hp = 1;
    while (hp < 8 && tiles * ((c->kv_heads + 2 * hp - 1) / (2 * hp)) >= 4 * sms) hp *= 2;
    while ((c->kv_heads + hp - 1) / hp > 65535) hp *= 2;
    P.heads_per_cta = hp;
    const dim3 grid((unsigned)tiles, (unsigned)((c->kv_heads + hp - 1) / hp));
    const bool bf = c->dtype == CB_BF16;
#define CB_KV4_CASE(d, g) \
    if (c->head_dim == d && c->group_size == g) \
        return bf ? launch_rows_t<__nv_bfloat16, d, g>(append, P, grid, stream) : launch_rows_t<__half, d, g>(append, P, grid, stream);
    CB_KV4_CASE(64, 32) CB_KV4_CASE(64, 64) CB_KV4_CASE(128, 32) CB_KV4_CASE(128, 64) CB_KV4_CASE(128, 128)
#undef CB_KV4_CASE
    set_error("kv4: no kernel for head_dim %d, group_size %d", c->head_dim, c->group_size);
    return CB_ERR_UNSUPPORTED;
}

int kv4_status_read_and_clear(int* out) {
    int v = 0, zero = 0;
    CB_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv4_status, sizeof(int)));
    CB_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int)));
    *out = v;
    return CB_OK;
}

}  // namespace cb
