// Writing to and reading from the 4-bit key/value cache (layout: cb_kv4.cuh).
//
//   lo = min(x), scale = round_T((max(x) - lo) / 15), code = round_half_even((x - lo) / scale) <= 15, value = code * scale + lo
//
// over the GS values x of a group, T the cache's 16-bit type.  A group with an infinity or a NaN keeps NaN for both and
// reads back as NaN; a scale below the smallest normal float is kept as 0, and the group reads back as lo.
//
// Both kernels are bound by memory: 2 bytes of a value on one side, 0.5 + 4 / GS on the other.  A CTA takes one block (16
// positions) of one sequence and a few heads, so that it looks up one page and owns every byte of the heads' blocks that
// tokens of this call fill; it turns them over in shared memory and moves whole blocks in 16-byte pieces.  A
// block that the call fills in part (a decode step's token, the ends of a prompt) is written value by value.  A thread
// owns 8 consecutive values of a row (token, head, K or V).
//
// Measured: 13584 tokens of 8 prompts, 32 heads, D = 128, are written in 79 us (3.6 TB/s; bfloat16, which meets more ties, 101 us), bound by the arithmetic of
// a value: issue slots are 73 % busy, DRAM 40 %.  54193 tokens of 8 heads are read back in 49.4 us (5.8 TB/s, near a copy's rate).  A decode step's append takes
// 3.4 us, little more than an empty launch.
#include <algorithm>

#include "cb_f32x2.cuh"
#include "cb_kv4.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeads = 8;          // heads of a CTA, at most
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

// n tokens from position p on lie in at most (n + 30) / 16 blocks.  Items are numbered with gaps, so that an item's sequence can be
// found without adding up the sequences' blocks: those of sequence b begin at cu[b] / 16 + 2 b (b * ((per_seq + 30) / 16)).
__host__ __device__ inline int64_t items_of(int64_t n_tokens, int64_t n_seqs, int64_t per_seq, bool packed) {
    return packed ? n_tokens / kKvBlock + 2 * n_seqs : n_seqs * ((per_seq + 30) / kKvBlock);
}

// What an item is: tokens [t0, t1) of the 16 positions of a block have their rows at packed token `token0` + position in the block.
struct Item {
    int64_t token0;
    int t0, t1, page, block;          // page < 0: nothing to do;  block inside its page
};
__device__ __forceinline__ Item find_item(const RowParams& P, int64_t idx) {
    Item it;
    it.page = -1; it.t0 = it.t1 = 0; it.token0 = 0; it.block = 0;
    int64_t b, k, first, n;
    if (P.cu != nullptr) {
        int64_t lo = 0, hi = P.n_seqs;            // the last sequence whose items begin at or before idx
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (max((int64_t)P.cu[mid], (int64_t)0) / kKvBlock + 2 * mid <= idx) lo = mid; else hi = mid;
        }
        b = lo;
        first = P.cu[b];
        n = P.cu[b + 1] - first;
        k = idx - (max(first, (int64_t)0) / kKvBlock + 2 * b);
    } else {
        const int64_t per = (P.per_seq + 30) / kKvBlock;
        b = idx / per;
        k = idx - b * per;
        first = b * P.per_seq;
        n = P.per_seq;
    }
    if (k < 0 || n <= 0 || first < 0 || first + n > P.n_tokens) return it;
    const int64_t start = P.starts[b], pos0 = ((start - (start & 15)) / kKvBlock + k) * kKvBlock;
    if (pos0 >= start + n) return it;
    it.t0 = (int)max(start - pos0, (int64_t)0);
    it.t1 = (int)min(start + n - pos0, (int64_t)kKvBlock);
    it.token0 = first + pos0 - start;
    const int64_t blk = pos0 / kKvBlock, row = blk / P.c.blocks_per_page;
    it.block = (int)(blk - row * P.c.blocks_per_page);
    const int64_t page = pos0 >= 0 && row < P.c.table_stride ? P.c.table[b * P.c.table_stride + row] : -1;
    if (page < 0 || page >= P.c.n_pages) atomicExch(&g_kv4_status, kKv4BadPage);
    else it.page = (int)page;
    return it;
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
    static constexpr float kTop = 65504.f;
    static constexpr uint32_t kTie = 0x1000u;                     // the bits of a float that a normal fp16 has not, half way between two
    // value = code * scale + lo with one rounding, for two codes at bits 0-3 and 16-19: 1024 + code from the bits, exactly
    __device__ static uint32_t values(uint32_t codes, uint32_t scale2, uint32_t lo2) {
        const uint32_t u = (codes & 0x000F000Fu) | 0x64006400u, k = 0x64006400u;
        const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&k));
        const __half2 r = __hfma2(c, *reinterpret_cast<const __half2*>(&scale2), *reinterpret_cast<const __half2*>(&lo2));
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
    static constexpr float kTop = 3.3895314e38f;
    static constexpr uint32_t kTie = 0x8000u;
    // as for fp16; 128 + code from the bits
    __device__ static uint32_t values(uint32_t codes, uint32_t scale2, uint32_t lo2) {
        const uint32_t u = (codes & 0x000F000Fu) | 0x43004300u, k = 0x43004300u;
        const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&k));
        const __nv_bfloat162 r = __hfma2(c, *reinterpret_cast<const __nv_bfloat162*>(&scale2), *reinterpret_cast<const __nv_bfloat162*>(&lo2));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

// What rounding took from d = a - b, exactly.
__device__ __forceinline__ float lost(float a, float b, float d) {
    const float bb = d - a;
    return (a - (d - bb)) - (b + bb);
}

// The group's (scale, lo) as stored, from its exact minimum and maximum.  The range hi - lo may need more bits than a float has; what it loses
// matters only where the quotient lies half way between two values of T.  (It lies there exactly if it looks so: 15 times such a value is a float, and
// other floats are at least a 2^-24th of it away, a quotient's rounding half as much at most.)  A range beyond the largest float is formed of halves,
// which are exact: a float holds half of any value of T.
constexpr float kWide = 2.2e37f;                                  // scales above it may have such a range: 15 of them are 3.3e38
template <typename T>
__device__ __forceinline__ uint32_t group_meta(float low, float hi) {
    const bool wide = Pair<T>::kTop > 15.f * kWide && hi - low == INFINITY && hi < INFINITY && low > -INFINITY;
    const float part = wide ? 0.5f : 1.f, lo = part * low;
    hi *= part;
    const float range = hi - lo;
    float q = __fdiv_rn(range, 15.0f);
    if ((__float_as_uint(q) & (2 * Pair<T>::kTie - 1)) == Pair<T>::kTie) {
        const float e = lost(hi, lo, range);
        if (e != 0.f) q = __uint_as_float(__float_as_uint(q) + (e > 0.f ? 1 : -1));
    }
    float scale = to_f32(from_f32<T>(q)), stored = low;
    if (wide) scale += scale;
    if (scale < 1.17549435e-38f) scale = 0.f;
    if (!(scale < INFINITY) || !(fabsf(low) < INFINITY)) scale = stored = __int_as_float(0x7fffffff);
    return Pair<T>::pack(scale, stored);
}

// Reciprocal to about 2^-22; what it gets wrong is found below.
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// round_half_even((x - lo) / scale), at most 15, for 8 bfloat16 values of a group whose range may be beyond the largest float: from halves.  Not inlined, since
// hardly ever called.
__device__ __noinline__ uint32_t wide_codes(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, float scale, float lo) {
    uint32_t word = 0u;
    const float step = 0.5f * scale, low = 0.5f * lo, h = 0.5f * step;
    for (int j = 0; j < 8; ++j) {
        const uint32_t two = j < 2 ? x0 : j < 4 ? x1 : j < 6 ? x2 : x3;
        const float v = 0.5f * __uint_as_float(j & 1 ? two & 0xFFFF0000u : two << 16), a = v - low;
        float c = floorf(__fdiv_rn(a, step));                     // the quotient's rounding up to a whole number: the remainder is then below 0
        float rest = fmaf(-c, step, a);
        if (rest < 0.f) { c -= 1.f; rest += step; }
        float past = rest - h;                                    // beyond half a step
        if (past == 0.f) past = lost(v, low, a);
        if (past == 0.f) past = (float)((int)c & 1);
        if (past > 0.f) c += 1.f;
        word |= (uint32_t)fminf(c, 15.f) << (4 * j);
    }
    return word;
}

// round_half_even((x - lo) / scale), at most 15, for 8 values: the codes as 4-bit fields.  Adding 1.5 * 2^23 rounds; the rounded
// quotients are gathered by multiply-adds.  The remainder a - code * scale of a = x - lo, which the fused multiply-add forms without rounding,
// shows where the approximate quotient met a tie or fell on the wrong side of one: there it is half a step or more (`half`: half a step, or 0
// where a code could exceed 15), and the eight are put right one by one.  (A tie in 8 values is met by 7 % of the warps for normal fp16
// values, by 38 % for bfloat16.)  a itself is rounded where x and lo are of very different size; that is less than the step in which remainders and half
// steps lie, so that it decides where the remainder is half a step and nowhere else.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const uint32_t (&x)[4], float scale, float lo, float inv, float half) {
    constexpr float kMagic = 12582912.f;
    const f32x2 minus_lo = pair(-lo, -lo), inv2 = pair(inv, inv), minus_scale = pair(-scale, -scale), magic = pair(kMagic, kMagic), back = pair(-kMagic, -kMagic);
    float c[8], rest[8], worst = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = Pair<T>::f2(x[j]);
        const f32x2 a = add2(pair(f.x, f.y), minus_lo), q = add2(fma2(a, inv2, magic), back);
        unpair(q, c[2 * j], c[2 * j + 1]);
        unpair(fma2(q, minus_scale, a), rest[2 * j], rest[2 * j + 1]);
        worst = fmaxf(worst, fmaxf(fabsf(rest[2 * j]), fabsf(rest[2 * j + 1])));
    }
    if (!(worst < half)) {
        if (!(scale > 0.f)) return 0u;                            // one value, or NaN
        if (Pair<T>::kTop > 15.f * kWide && scale > kWide) return wide_codes(x[0], x[1], x[2], x[3], scale, lo);
        const float h = 0.5f * scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float past = fabsf(rest[j]) - h;                      // beyond half a step, in the remainder's direction
            if (past == 0.f) {
                const float2 f = Pair<T>::f2(x[j / 2]);
                const float v = j & 1 ? f.y : f.x;
                past = copysignf(1.f, rest[j]) * lost(v, lo, v - lo);
                if (past == 0.f) past = (float)((int)c[j] & 1);   // a tie: to even
            }
            if (past > 0.f) c[j] += copysignf(1.f, rest[j]);
            c[j] = fminf(c[j], 15.f);
        }
    }
    const float p = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]) + kMagic;
    const float q = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]) + kMagic;
    return __byte_perm(__float_as_uint(p), __float_as_uint(q), 0x5410);
}

// Where thread `tid` stands: 8 values from `d` on, of block position `tok`, in every kPer-th row from `sub` on.
template <int D> struct Place {
    static constexpr int kTpr = D / 8;                                     // threads of a row
    static constexpr int kPer = kThreads / (kTpr * kKvBlock);              // rows of a token side by side: 1 at D = 128, 2 at 64
};

template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads, 4)              // 64 registers; with three CTAs to an SM writing and reading 13584 tokens takes 136 us for 125
kv4_append_kernel(const RowParams P) {
    using L = KvLayout<D, GS>;
    constexpr int kTpr = Place<D>::kTpr, kPer = Place<D>::kPer, kBatch = 4;       // kBatch: loads in flight
    __shared__ __align__(16) unsigned char image[kMaxHeads][L::kBytes];
    const Item it = find_item(P, blockIdx.x);
    if (it.page < 0) return;
    const int tid = threadIdx.x;
    const int d = tid % kTpr * 8, tok = (tid / kTpr) % kKvBlock, sub = tid / (kTpr * kKvBlock);
    const int h0 = blockIdx.y * P.heads_per_cta, heads = min(P.heads_per_cta, P.c.kv_heads - h0), rows = 2 * heads;      // a row: (head, K or V)
    const bool live = tok >= it.t0 && tok < it.t1, full = it.t1 - it.t0 == kKvBlock, lead = d % GS == 0;
    const int64_t token = it.token0 + tok;
    const int64_t stride = (int64_t)P.c.blocks_per_page * L::kBytes;              // from a head to the next
    unsigned char* first = P.c.pages + (((int64_t)it.page * P.c.kv_heads + h0) * P.c.blocks_per_page + it.block) * L::kBytes;
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
                x[i] = __ldg(reinterpret_cast<const uint4*>(src + d));
            }
        }
        // All lanes take part in the shuffles; what dead ones compute is dropped.  Groups' (min, -max) first, of all the rows; then each
        // lane of a group finishes one row's, and they are passed around.
        uint32_t both[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            uint32_t mn = Pair<T>::min2(Pair<T>::min2(x[i].x, x[i].y), Pair<T>::min2(x[i].z, x[i].w));
            uint32_t mx = Pair<T>::max2(Pair<T>::max2(x[i].x, x[i].y), Pair<T>::max2(x[i].z, x[i].w)) ^ 0x80008000u;
            both[i] = Pair<T>::min2(__byte_perm(mn, mx, 0x5410), __byte_perm(mn, mx, 0x7632));
        }
#pragma unroll
        for (int o = 1; o < GS / 8; o <<= 1)
#pragma unroll
            for (int i = 0; i < kBatch; ++i) both[i] = Pair<T>::min2(both[i], __shfl_xor_sync(0xffffffffu, both[i], o));
        static_assert(kBatch == 4 && GS / 8 >= 4, "a lane for each row");
        const float2 mm = Pair<T>::f2(tid & 2 ? (tid & 1 ? both[3] : both[2]) : (tid & 1 ? both[1] : both[0]));
        const uint32_t my_meta = group_meta<T>(mm.x, -mm.y);
        const float my_scale = Pair<T>::f2(my_meta).x, my_inv = rcp_approx(my_scale);
        // the rounding of a scale of few bits can carry the largest value past 15.5 steps; NaN fails the comparison
        const float my_half = -mm.y - mm.x < 15.4f * my_scale ? 0.5f * my_scale : 0.f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i * kPer, from = (tid & 31 & ~3) | i;
            const uint32_t meta = __shfl_sync(0xffffffffu, my_meta, from);
            const float inv = __shfl_sync(0xffffffffu, my_inv, from), half = __shfl_sync(0xffffffffu, my_half, from);
            const float2 sl = Pair<T>::f2(meta);
            const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            const uint32_t word = codes_of<T>(xs, sl.x, sl.y, inv, half);
            if (!live || r >= rows) continue;
            unsigned char* blk = full ? image[r >> 1] : first + (r >> 1) * stride;
            if ((r & 1) == 0) {
                *reinterpret_cast<uint32_t*>(blk + tok * L::kRow + L::k_nibble(d) / 2) = word;
                if (lead) *reinterpret_cast<uint32_t*>(blk + L::kKMeta + tok * L::kMeta + (d / GS) * 4) = meta;
            } else {
                *reinterpret_cast<uint16_t*>(blk + L::kVCodes + L::v_byte(d, tok)) = (uint16_t)word;
                *reinterpret_cast<uint16_t*>(blk + L::kVCodes + L::v_byte(d + 4, tok)) = (uint16_t)(word >> 16);
                if (lead) *reinterpret_cast<uint32_t*>(blk + L::kVMeta + tok * L::kMeta + (d / GS) * 4) = meta;
            }
        }
    }
    if (!full) return;
    __syncthreads();
    constexpr int kPieces = L::kBytes / 16;
    for (int i = tid; i < heads * kPieces; i += kThreads) {
        const int h = i / kPieces, at = i % kPieces * 16;
        *reinterpret_cast<uint4*>(first + h * stride + at) = *reinterpret_cast<const uint4*>(image[h] + at);
    }
}

template <typename T, int D, int GS>
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const RowParams P) {
    using L = KvLayout<D, GS>;
    constexpr int kTpr = Place<D>::kTpr, kPer = Place<D>::kPer;
    __shared__ __align__(16) unsigned char image[kMaxHeads][L::kBytes];
    const Item it = find_item(P, blockIdx.x);
    if (it.page < 0) return;
    const int tid = threadIdx.x;
    const int d = tid % kTpr * 8, tok = (tid / kTpr) % kKvBlock, sub = tid / (kTpr * kKvBlock);
    const int h0 = blockIdx.y * P.heads_per_cta, heads = min(P.heads_per_cta, P.c.kv_heads - h0);
    const int64_t stride = (int64_t)P.c.blocks_per_page * L::kBytes;
    const unsigned char* first = P.c.pages + (((int64_t)it.page * P.c.kv_heads + h0) * P.c.blocks_per_page + it.block) * L::kBytes;
    constexpr int kPieces = L::kBytes / 16;
    for (int i = tid; i < heads * kPieces; i += kThreads) {
        const int h = i / kPieces, at = i % kPieces * 16;
        *reinterpret_cast<uint4*>(image[h] + at) = __ldcs(reinterpret_cast<const uint4*>(first + h * stride + at));
    }
    __syncthreads();
    if (tok < it.t0 || tok >= it.t1) return;
    const int64_t out = ((it.token0 + tok) * P.c.kv_heads + h0) * D + d;
    for (int r = sub; r < 2 * heads; r += kPer) {
        const unsigned char* blk = image[r >> 1];
        uint32_t word, meta;
        if ((r & 1) == 0) {
            word = *reinterpret_cast<const uint32_t*>(blk + tok * L::kRow + L::k_nibble(d) / 2);
            meta = *reinterpret_cast<const uint32_t*>(blk + L::kKMeta + tok * L::kMeta + (d / GS) * 4);
        } else {
            word = *reinterpret_cast<const uint16_t*>(blk + L::kVCodes + L::v_byte(d, tok)) |
                   ((uint32_t)*reinterpret_cast<const uint16_t*>(blk + L::kVCodes + L::v_byte(d + 4, tok)) << 16);
            meta = *reinterpret_cast<const uint32_t*>(blk + L::kVMeta + tok * L::kMeta + (d / GS) * 4);
        }
        const uint32_t scale2 = __byte_perm(meta, 0u, 0x1010), lo2 = __byte_perm(meta, 0u, 0x3232);
        uint32_t y[4];                                            // values 0 and 4, 1 and 5, 2 and 6, 3 and 7
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = Pair<T>::values(word >> (4 * j), scale2, lo2);
        const float2 sl = Pair<T>::f2(meta);
        if (fmaf(15.f, sl.x, sl.y) > Pair<T>::kTop) {
            // the rounding of scale can carry the largest values of such a group past the type's largest number: they are that number
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = fmaf((float)((word >> (4 * j)) & 15u), sl.x, sl.y), b = fmaf((float)((word >> (4 * j + 16)) & 15u), sl.x, sl.y);
                y[j] = Pair<T>::pack(fminf(a, Pair<T>::kTop), fminf(b, Pair<T>::kTop));
            }
        }
        const uint32_t o[4] = {__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                               __byte_perm(y[2], y[3], 0x7632)};
        T* dst = ((r & 1) ? reinterpret_cast<T*>(P.v_out) : reinterpret_cast<T*>(P.k_out)) + out + (r >> 1) * D;
        __stcs(reinterpret_cast<uint4*>(dst), make_uint4(o[0], o[1], o[2], o[3]));
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
    // few blocks: one head to a CTA, so that a decode step spreads over the SMs; many: up to eight, for fewer look-ups and more loads in flight (13584 tokens
    // written and read 122 us, one head to a CTA 276; 54193 read 49 and 88.5)
    const int64_t items = items_of(n_tokens, n_seqs, P.per_seq, cu != nullptr);
    int hp = 1;
    while (hp < kMaxHeads && items * ((c->kv_heads + 2 * hp - 1) / (2 * hp)) >= 4 * sms) hp *= 2;
    P.heads_per_cta = hp;
    const int64_t head_ctas = (c->kv_heads + hp - 1) / hp;
    if (items >= (1ll << 31) || head_ctas > 65535) { set_error("kv4: too many tokens, sequences or heads in one call"); return CB_ERR_INVALID; }
    const dim3 grid((unsigned)items, (unsigned)head_ctas);
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
