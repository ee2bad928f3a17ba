// Attention of the newest tokens of each sequence over the 4-bit key/value cache (layout: cb_kv4.cuh).
//
// For one sequence and key head, with n cached tokens and R = new tokens * query heads per key head rows q_r:
//   x_rt = c * q_r . k_t,  k_t = code * scale + lo  by groups j   =>   x_rt = c * sum_j (scale_tj * (q_rj . code_tj) + lo_tj * sum(q_rj))
//   p_rt = exp(x_rt - max),  out_r = sum_t p_rt v_t / sum_t p_rt  =>   out_rd = (sum_t (p_rt scale_tj) code_td + sum_t p_rt lo_tj) / sum_t p_rt
// so both products run on the bare codes, and scale and lo enter per (token, group), not per value.
//
// What bounds it: the cache is read once, D / 2 + 4 D / GS bytes for the keys of a token and head and the same for its values.  At
// the memory's rate an SM has about 2.8 lane instructions for each code, so the codes go to the tensor cores (mma.sync
// m16n8k16, fp16) as they are: a masked 4-bit field at bits 0-3 of an fp16 is the subnormal code * 2^-24, at bits 4-7
// code * 2^-20; one AND makes two operands.  Codes are the 16-row operand (S^T = K q^T, O^T = V^T P^T), query rows the 8
// columns, so that a step of 16 x 16 codes is one instruction whatever the number of rows; P^T gets from the first product's
// accumulator layout into the second's operand layout by movmatrix.  (tcgen05 would need the codes expanded to 8 or 16 bits in
// shared or tensor memory, which costs more than the product.)
//
// Precision: q_r is scaled by a power of two so that its largest value lies in [2^13, 2^14) and then rounded to fp16: exact for
// fp16 inputs down to 2^-24 of the row's largest value, and for bfloat16 inputs alike.  p * scale is scaled by a power of two so
// that scale's part lies in [2^14, 2^15) for the largest scale met and then rounded to fp16 (relative error 2^-11; below 2^-28
// of the largest possible weight absolute).  All sums, the softmax statistics and the lo part are fp32.
//
// Work: the 16-token blocks of all (sequence, row tile, key head) segments form one line that is cut into equal parts, one for each CTA (two to an
// SM), whatever the lengths are; lengths are read on the device, so a captured launch serves any.  The 8 warps of a CTA take
// pairs of blocks in turn, each with a ring of its own filled by bulk copies (one per block), and keep running maxima, sums and
// outputs of their own; they meet in shared memory at the end of a segment.  Where a segment is cut, its parts leave
// (max, sum, output) in scratch and the CTA that arrives last adds them in order of position: the result does not
// depend on timing.
#include <algorithm>

#include "cb_kv4.cuh"

namespace cb {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kStageBlocks = 2;                       // blocks of a ring slot
constexpr long long kWaitCycles = 2000000000ll;       // about a second

__device__ int g_kv4_attn_status;

struct AttnParams {
    Kv4View c;
    const void* q; int64_t q_b, q_t, q_h;             // strides in elements
    void* out;                                        // [B, T, H, D]
    const int32_t* lengths;
    int64_t B;
    int T, H, G, R, row_tiles;
    float scale_log2;                                 // softmax scale * log2(e)
    int* counters;                                    // [B * kv_heads * row_tiles], zero between calls
    float* partial;                                   // [grid][2][rows of a tile * (D + 2)]
};

template <int D, int GS, int NT>
struct AttnCfg {
    using L = KvLayout<D, GS>;
    static constexpr int kRows = 8 * NT;
    static constexpr int kSlotBytes = kStageBlocks * L::kBytes;
    static constexpr int kCtasPerSm = NT == 1 ? 2 : 1;
    // the ring fills what an SM has; the slots of a warp are at most 8
    static constexpr int kRingBudget = (NT == 1 ? 108 : 216) * 1024;
    static constexpr int kSlots = kRingBudget / (kWarps * kSlotBytes) > 8 ? 8 : kRingBudget / (kWarps * kSlotBytes);
    static constexpr int kRing = kWarps * kSlots * kSlotBytes;
    static constexpr int kMerge = kWarps * kRows * D * 4;             // reuses the ring's space
    static_assert(kMerge <= kRing, "the merge buffer lies over the ring");
    static constexpr int kStatsOff = kRing;                           // [2][kWarps][kRows] floats: max, sum
    static constexpr int kBarOff = kStatsOff + 2 * kWarps * kRows * 4;
    static constexpr int kOkOff = kBarOff + kWarps * kSlots * 8;      // [kWarps][kSlots] blocks whose page is good
    static constexpr int kMiscOff = kOkOff + kWarps * kSlots * 4;
    static constexpr int kSmem = kMiscOff + 64 + kWarps * 8;
    static_assert(kSmem <= (227 * 1024) / kCtasPerSm - 1024, "shared memory of an SM");
    static constexpr int kPartFloats = kRows * (D + 2);
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    for (;;) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (clock64() - t0 > kWaitCycles) return false;
    }
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
template <int N> __device__ __forceinline__ void lds_words(const unsigned char* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

__device__ __forceinline__ int64_t seq_len(const AttnParams& P, int64_t b) {
    const int64_t cap = P.c.table_stride * P.c.blocks_per_page * kKvBlock;
    return min(max((int64_t)P.lengths[b], (int64_t)0), cap);
}
__device__ __forceinline__ int64_t seq_blocks(const AttnParams& P, int64_t b) { return (seq_len(P, b) + kKvBlock - 1) / kKvBlock; }

template <typename T, int D, int GS, int NT>
__global__ void __launch_bounds__(kThreads, (AttnCfg<D, GS, NT>::kCtasPerSm))
kv4_attention_kernel(const AttnParams P) {
    using C = AttnCfg<D, GS, NT>;
    using L = typename C::L;
    constexpr int NG = L::NG, kSlots = C::kSlots, kRows = C::kRows;
    constexpr int KW = D / 32, KWG = GS / 32;          // code words of a lane and key row, of one group
    constexpr int VW = D / 64;                         // code words of a lane and value row
    extern __shared__ __align__(128) unsigned char smem[];
    float* merge = reinterpret_cast<float*>(smem);
    float* st_max = reinterpret_cast<float*>(smem + C::kStatsOff);
    float* st_sum = st_max + kWarps * kRows;
    volatile int* misc = reinterpret_cast<volatile int*>(smem + C::kMiscOff);           // [0] abort, [1] last arrival
    int64_t* red = reinterpret_cast<int64_t*>(smem + C::kMiscOff + 64);                 // [kWarps]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bars = smem_u32(smem + C::kBarOff) + warp * kSlots * 8;
    volatile uint32_t* slot_ok = reinterpret_cast<volatile uint32_t*>(smem + C::kOkOff) + warp * kSlots;
    unsigned char* ring = smem + (size_t)warp * kSlots * C::kSlotBytes;
    const uint32_t ring_u32 = smem_u32(ring);
    const int kv_heads = P.c.kv_heads, segs = kv_heads * P.row_tiles;

    if (lane == 0) {
        for (int s = 0; s < kSlots; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * s));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 0) misc[0] = 0;

    // ---- the whole line's length, and sequences without keys: their rows are zero
    int64_t blocks = 0;
    for (int64_t b = tid; b < P.B; b += kThreads) blocks += seq_blocks(P, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) blocks += __shfl_xor_sync(0xffffffffu, blocks, o);
    if (lane == 0) red[warp] = blocks;
    for (int64_t b = blockIdx.x; b < P.B; b += gridDim.x)
        if (seq_blocks(P, b) == 0) {
            uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(P.out) + b * P.T * P.H * D);
            for (int i = tid; i < P.T * P.H * D / 2; i += kThreads) o[i] = 0u;
        }
    __syncthreads();
    int64_t U = 0;
    for (int w = 0; w < kWarps; ++w) U += red[w];
    U *= segs;
    const int64_t nc = min((int64_t)gridDim.x, U);
    if (blockIdx.x >= nc) return;
    const int64_t u0 = blockIdx.x * U / nc, u1 = (blockIdx.x + 1) * U / nc;

    // ---- the sequence that holds unit u0 (every warp for itself)
    int64_t b = 0, base = 0, nb = 0;
    for (int64_t b0 = 0; b0 < P.B; b0 += 32) {
        const int64_t mine = b0 + lane < P.B ? seq_blocks(P, b0 + lane) * segs : 0;
        int64_t cum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, cum, o);
            if (lane >= o) cum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + cum > u0);
        if (past != 0u) {
            const int l = __ffs(past) - 1;
            b = b0 + l;
            nb = __shfl_sync(0xffffffffu, mine, l) / segs;
            base += __shfl_sync(0xffffffffu, cum - mine, l);
            break;
        }
        base += __shfl_sync(0xffffffffu, cum, 31);
    }

    uint32_t it = 0;                                   // stages this warp has taken from its ring, ever
    for (int64_t u = u0; u < u1;) {
        while (u >= base + nb * segs) {
            base += nb * segs;
            if (++b >= P.B) return;                    // only if lengths changed while the kernel ran
            nb = seq_blocks(P, b);
        }
        const int seg = (int)((u - base) / nb);
        const int64_t seg0 = base + seg * nb;          // first unit of the segment
        const int64_t blk0 = u - seg0, blk1 = min(nb, u1 - seg0);
        const int kvh = seg % kv_heads, row0 = (seg / kv_heads) * kRows;
        const int len = (int)min(seq_len(P, b), (int64_t)0x7fffffff);

        // ---- query rows: fp16 fragments, their scales, sums and limits
        uint32_t qf[NT][KW * 4];
        float qsum[NT][NG][2], qmul[NT][2];
        int lim[NT][2], lim_min = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row0 + n * 8 + g;
            const bool live = r < P.R;
            const int rt = live ? r / P.G : 0, rg = live ? r % P.G : 0;
            const T* src = reinterpret_cast<const T*>(P.q) + b * P.q_b + rt * P.q_t + (int64_t)(kvh * P.G + rg) * P.q_h;
            float x[KW][8], mx = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const int d0 = (w / KWG) * GS + t * (GS / 4) + (w % KWG) * 8;
                const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(src + d0)) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<T>(vs[i]);
                    x[w][2 * i] = f.x; x[w][2 * i + 1] = f.y;
                    mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = min(max((int)(__float_as_uint(mx) >> 23), 14), 254);
            const float f = __uint_as_float((uint32_t)(267 - e) << 23);              // 2^(140 - e)
            float sum[NG];
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                float h[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = __half2float(__float2half_rn(x[w][i] * f));
                qf[n][4 * w + 0] = pack_h2(h[0], h[4]);
                qf[n][4 * w + 1] = pack_h2(h[1] * 0.0625f, h[5] * 0.0625f);          // meets codes * 2^-20
                qf[n][4 * w + 2] = pack_h2(h[2], h[6]);
                qf[n][4 * w + 3] = pack_h2(h[3] * 0.0625f, h[7] * 0.0625f);
                const float part = ((h[0] + h[1]) + (h[2] + h[3])) + ((h[4] + h[5]) + (h[6] + h[7]));
                if (w % KWG == 0) sum[w / KWG] = part; else sum[w / KWG] += part;
            }
            const float mul = P.scale_log2 * __uint_as_float((uint32_t)(e - 13) << 23) * 16777216.f;
            const int limit = live ? len - P.T + 1 + rt : 0;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
                sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
                sum[j] *= 5.9604644775390625e-8f;                                    // 2^-24, as the products with codes
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {                                            // columns 2t, 2t + 1 of the accumulators
                const int from = (2 * t + c) * 4;
#pragma unroll
                for (int j = 0; j < NG; ++j) qsum[n][j][c] = __shfl_sync(0xffffffffu, sum[j], from);
                qmul[n][c] = __shfl_sync(0xffffffffu, mul, from);
                lim[n][c] = __shfl_sync(0xffffffffu, limit, from);
                lim_min = min(lim_min, lim[n][c]);
            }
        }
        lim_min = __reduce_min_sync(0xffffffffu, lim_min);

        float o[NT][D / 16][4], m_run[NT][2], l_run[NT][2], z[NT][NG][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m_run[n][c] = -INFINITY; l_run[n][c] = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) z[n][j][c] = 0.f;
            }
        }
        int s_exp = 15;                                // exponent field of the power of two that p * scale is divided by

        // ---- this warp's stages of the piece: stage i holds blocks first(i) .. + cnt; few blocks: one to a stage
        const int pieces = (int)(blk1 - blk0);
        const int per = pieces > kWarps ? kStageBlocks : 1;
        const int nstage = (pieces + per - 1) / per;
        const int mine = warp < nstage ? (nstage - 1 - warp) / kWarps + 1 : 0;
        auto issue = [&](int i, uint32_t at) {
            const uint32_t s = at % kSlots;
            const int64_t first = blk0 + (int64_t)(warp + i * kWarps) * per;
            const int64_t blk = first + lane;
            int64_t page = -1;
            const bool in = lane < per && blk < blk1;
            if (in) {
                page = P.c.table[b * P.c.table_stride + blk / P.c.blocks_per_page];
                if (page < 0 || page >= P.c.n_pages) { page = -1; atomicExch(&g_kv4_attn_status, kKv4BadPage); }
            }
            const unsigned good = __ballot_sync(0xffffffffu, page >= 0);
            const uint32_t bar = bars + 8 * s;
            if (lane == 0) {
                slot_ok[s] = good;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)(__popc(good) * L::kBytes)) : "memory");
            }
            __syncwarp();
            if (page >= 0) {
                const unsigned char* src = P.c.pages + ((page * kv_heads + kvh) * P.c.blocks_per_page + blk % P.c.blocks_per_page) * L::kBytes;
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(ring_u32 + s * C::kSlotBytes + lane * L::kBytes), "l"(src), "r"((uint32_t)L::kBytes), "r"(bar) : "memory");
            }
        };
        for (int i = 0; i < kSlots && i < mine; ++i) issue(i, it + i);

        const int ra = g & 1 ? 7 - (g >> 1) : (g >> 1);            // token of accumulator row g; row g + 8 is token ra + 8
        for (int i = 0; i < mine; ++i) {
            const uint32_t at = it + i, s = at % kSlots;
            if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * s, (at / kSlots) & 1))) {
                if (lane == 0) { misc[0] = 1; atomicExch(&g_kv4_attn_status, kKv4Wait); }
                for (int k = i + 1; k < mine && k < i + kSlots; ++k) mbar_wait(bars + 8 * ((it + k) % kSlots), ((it + k) / kSlots) & 1);
                break;
            }
            const int64_t first = blk0 + (int64_t)(warp + i * kWarps) * per;
            const unsigned good = slot_ok[s];
            const unsigned char* stage = ring + s * C::kSlotBytes;
            const int cnt = (int)min((int64_t)per, blk1 - first);
            // every token of the stage seen by every row?
            const bool plain = good == (1u << cnt) - 1u && cnt == kStageBlocks && (first + cnt) * kKvBlock <= lim_min;

            float x[kStageBlocks][NT][4];
            float mx[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) mx[n][0] = mx[n][1] = -INFINITY;
            float smax = 0.f;
#pragma unroll
            for (int k = 0; k < kStageBlocks; ++k) {
                const bool there = (good >> k) & 1u;
                if (!there) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) x[k][n][0] = x[k][n][1] = x[k][n][2] = x[k][n][3] = -INFINITY;
                    continue;
                }
                const unsigned char* blk = stage + k * L::kBytes;
                uint32_t wa[KW], wb[KW], ma[NG], mb[NG];
                lds_words<KW>(blk + ra * L::kRow + t * (D / 8), wa);
                lds_words<KW>(blk + (ra + 8) * L::kRow + t * (D / 8), wb);
                lds_words<NG>(blk + L::kKMeta + ra * L::kMeta, ma);
                lds_words<NG>(blk + L::kKMeta + (ra + 8) * L::kMeta, mb);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    float acc[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
                    for (int w = j * KWG; w < (j + 1) * KWG; ++w) {
                        const uint32_t ya = wa[w] >> 8, yb = wb[w] >> 8;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816(acc[n], wa[w] & 0x000F000Fu, wb[w] & 0x000F000Fu, wa[w] & 0x00F000F0u, wb[w] & 0x00F000F0u,
                                     qf[n][4 * w], qf[n][4 * w + 1]);
                            mma16816(acc[n], ya & 0x000F000Fu, yb & 0x000F000Fu, ya & 0x00F000F0u, yb & 0x00F000F0u,
                                     qf[n][4 * w + 2], qf[n][4 * w + 3]);
                        }
                    }
                    const float2 sa = unpack2<T>(ma[j]), sb = unpack2<T>(mb[j]);     // (scale, lo)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float va = fmaf(acc[n][c], sa.x, sa.y * qsum[n][j][c]);
                            const float vb = fmaf(acc[n][2 + c], sb.x, sb.y * qsum[n][j][c]);
                            x[k][n][c] = j == 0 ? va : x[k][n][c] + va;
                            x[k][n][2 + c] = j == 0 ? vb : x[k][n][2 + c] + vb;
                        }
                }
                const int tok = (int)(first + k) * kKvBlock + ra;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        x[k][n][c] *= qmul[n][c];
                        x[k][n][2 + c] *= qmul[n][c];
                        if (!plain) {
                            if (tok >= lim[n][c]) x[k][n][c] = -INFINITY;
                            if (tok + 8 >= lim[n][c]) x[k][n][2 + c] = -INFINITY;
                        }
                        mx[n][c] = fmaxf(mx[n][c], fmaxf(x[k][n][c], x[k][n][2 + c]));
                    }
                uint32_t va[NG], vb[NG];
                lds_words<NG>(blk + L::kVMeta + ra * L::kMeta, va);
                lds_words<NG>(blk + L::kVMeta + (ra + 8) * L::kMeta, vb);
#pragma unroll
                for (int j = 0; j < NG; ++j) {                       // fmaxf drops NaN
                    const float s0 = unpack2<T>(va[j]).x, s1 = unpack2<T>(vb[j]).x;
                    smax = fmaxf(smax, plain || tok < len ? s0 : 0.f);
                    smax = fmaxf(smax, plain || tok + 8 < len ? s1 : 0.f);
                }
            }
            // ---- running maximum and scale reference
            float alpha[NT][2];
            const int e_new = max(s_exp, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(smax)) >> 23));
            bool moved = e_new != s_exp;
            const float rs = __uint_as_float((uint32_t)max(127 + s_exp - e_new, 0) << 23);
            s_exp = e_new;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = mx[n][c];
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    const float mn = fmaxf(m_run[n][c], m);
                    alpha[n][c] = mn == m_run[n][c] ? 1.f : ex2(m_run[n][c] - mn);
                    moved = moved || alpha[n][c] != 1.f;
                    m_run[n][c] = mn;
                }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        l_run[n][c] *= alpha[n][c];
#pragma unroll
                        for (int j = 0; j < NG; ++j) z[n][j][c] *= alpha[n][c];
                        alpha[n][c] *= rs;
                    }
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        o[n][d][0] *= alpha[n][0]; o[n][d][1] *= alpha[n][1];
                        o[n][d][2] *= alpha[n][0]; o[n][d][3] *= alpha[n][1];
                    }
                }
            }
            const float cmul = __uint_as_float((uint32_t)(268 - s_exp) << 23);       // 2^14 / 2^(s_exp - 127)
#pragma unroll
            for (int k = 0; k < kStageBlocks; ++k) {
                if (!((good >> k) & 1u)) continue;
                const unsigned char* blk = stage + k * L::kBytes;
                uint32_t va[NG], vb[NG];
                lds_words<NG>(blk + L::kVMeta + ra * L::kMeta, va);
                lds_words<NG>(blk + L::kVMeta + (ra + 8) * L::kMeta, vb);
                float p[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float m = m_run[n][c] == -INFINITY ? 0.f : m_run[n][c];
                        p[n][c] = ex2(x[k][n][c] - m);
                        p[n][2 + c] = ex2(x[k][n][2 + c] - m);
                        l_run[n][c] += p[n][c] + p[n][2 + c];
                    }
                uint32_t pb[NT][NG][2];
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const float2 sa = unpack2<T>(va[j]), sb = unpack2<T>(vb[j]);
                    const float fa = sa.x * cmul, fb = sb.x * cmul;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float h[4] = {p[n][0] * fa, p[n][1] * fa, p[n][2] * fb, p[n][3] * fb};
                        float y[4] = {p[n][0] * sa.y, p[n][1] * sa.y, p[n][2] * sb.y, p[n][3] * sb.y};
                        if (!plain) {
                            // what a row does not see adds nothing, whatever is stored there
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (p[n][c] == 0.f) h[c] = y[c] = 0.f;
                        }
                        z[n][j][0] += y[0] + y[2];
                        z[n][j][1] += y[1] + y[3];
                        pb[n][j][0] = movmatrix_t(pack_h2(h[0], h[1]));
                        pb[n][j][1] = movmatrix_t(pack_h2(h[2], h[3]));
                    }
                }
                // tokens t, 7 - t, t + 8, 15 - t: columns 2t, 2t + 1, 2t + 8, 2t + 9 of the operand
                uint32_t v[4][VW];
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const int tk = (i4 & 1 ? 7 - t : t) + (i4 & 2 ? 8 : 0);
                    const int at_byte = D == 128 ? (g * 8) ^ (((tk >> 1) & 1) << 5) : g * 4;
                    lds_words<VW>(blk + L::kVCodes + tk * L::kRow + at_byte, v[i4]);
                }
#pragma unroll
                for (int hw = 0; hw < 2 * VW; ++hw) {                                // four values of this lane
                    const int j = hw * 4 / (GS / 8);
                    const uint32_t x0 = __byte_perm(v[0][hw >> 1], v[1][hw >> 1], hw & 1 ? 0x7632 : 0x5410);
                    const uint32_t x1 = __byte_perm(v[2][hw >> 1], v[3][hw >> 1], hw & 1 ? 0x7632 : 0x5410);
                    const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816(o[n][2 * hw], x0 & 0x000F000Fu, y0 & 0x000F000Fu, x1 & 0x000F000Fu, y1 & 0x000F000Fu, pb[n][j][0], pb[n][j][1]);
                        mma16816(o[n][2 * hw + 1], x0 & 0x00F000F0u, y0 & 0x00F000F0u, x1 & 0x00F000F0u, y1 & 0x00F000F0u, pb[n][j][0], pb[n][j][1]);
                    }
                }
            }
            __syncwarp();
            if (i + kSlots < mine) issue(i + kSlots, at + kSlots);       // every code of this slot has gone into a product
        }
        it += mine;

        // ---- the warps' results meet: value = o * 2^24 (2^20) / cmul + z
        __syncthreads();                                                // nobody reads its ring any more
        {
            const float back = __uint_as_float((uint32_t)(s_exp - 14) << 23);        // 1 / cmul
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float zz[NG], l = l_run[n][c];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        zz[j] = z[n][j][c];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) zz[j] += __shfl_xor_sync(0xffffffffu, zz[j], d);
                    }
                    const int row = n * 8 + 2 * t + c;
                    if (g == 0) { st_max[warp * kRows + row] = m_run[n][c]; st_sum[warp * kRows + row] = l; }
                    float* dst = merge + ((size_t)warp * kRows + row) * D;
#pragma unroll
                    for (int hw = 0; hw < 2 * VW; ++hw) {
                        const int j = hw * 4 / (GS / 8);
                        const int d = j * GS + g * (GS / 8) + (hw * 4) % (GS / 8);
                        float4 r4;
                        r4.x = fmaf(o[n][2 * hw][c] * 16777216.f, back, zz[j]);
                        r4.y = fmaf(o[n][2 * hw + 1][c] * 1048576.f, back, zz[j]);
                        r4.z = fmaf(o[n][2 * hw][2 + c] * 16777216.f, back, zz[j]);
                        r4.w = fmaf(o[n][2 * hw + 1][2 + c] * 1048576.f, back, zz[j]);
                        *reinterpret_cast<float4*>(dst + d) = r4;
                    }
                }
            }
        }
        __syncthreads();
        if (misc[0] != 0) return;
        const bool whole = blk0 == 0 && blk1 == nb;
        auto store = [&](int row, int d, float2 v, float l) {           // two neighbouring values of a finished row
            const int r = row0 + row;
            if (r >= P.R) return;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (l == 0.f) v = make_float2(0.f, 0.f);
            T* dst = reinterpret_cast<T*>(P.out) + ((b * P.T + r / P.G) * P.H + kvh * P.G + r % P.G) * D + d;
            dst[0] = from_f32<T>(v.x * inv);
            dst[1] = from_f32<T>(v.y * inv);
        };
        float* my_part = P.partial + ((int64_t)blockIdx.x * 2 + (u == u0 ? 0 : 1)) * C::kPartFloats;
        for (int idx = tid; idx < kRows * D / 2; idx += kThreads) {
            const int row = idx / (D / 2), d = idx % (D / 2) * 2;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, st_max[w * kRows + row]);
            float2 v = make_float2(0.f, 0.f);
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = st_max[w * kRows + row] == -INFINITY ? 0.f : ex2(st_max[w * kRows + row] - m);
                if (f != 0.f) {
                    const float2 a = *reinterpret_cast<const float2*>(merge + ((size_t)w * kRows + row) * D + d);
                    v.x = fmaf(f, a.x, v.x); v.y = fmaf(f, a.y, v.y);
                    l = fmaf(f, st_sum[w * kRows + row], l);
                }
            }
            if (whole) store(row, d, v, l);
            else {
                *reinterpret_cast<float2*>(my_part + row * D + d) = v;
                if (d == 0) { my_part[kRows * D + row] = m; my_part[kRows * D + kRows + row] = l; }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            const int64_t c0 = ((seg0 + 1) * nc - 1) / U, c1 = ((seg0 + nb) * nc - 1) / U;      // CTAs that hold its first and last unit
            if (tid == 0) {
                int* counter = P.counters + b * segs + seg;
                const bool last = atomicAdd(counter, 1) == (int)(c1 - c0);
                if (last) *counter = 0;
                __threadfence();
                misc[1] = last;
            }
            __syncthreads();
            if (misc[1] != 0) {
                const float* first_part = P.partial + (c0 * 2 + (c0 * U / nc == seg0 ? 0 : 1)) * C::kPartFloats;
                for (int idx = tid; idx < kRows * D / 2; idx += kThreads) {
                    const int row = idx / (D / 2), d = idx % (D / 2) * 2;
                    float m = -INFINITY;
                    for (int64_t c = c0; c <= c1; ++c) {
                        const float* part = c == c0 ? first_part : P.partial + c * 2 * C::kPartFloats;
                        m = fmaxf(m, __ldcg(part + kRows * D + row));
                    }
                    float2 v = make_float2(0.f, 0.f);
                    float l = 0.f;
                    for (int64_t c = c0; c <= c1; ++c) {
                        const float* part = c == c0 ? first_part : P.partial + c * 2 * C::kPartFloats;
                        const float pm = __ldcg(part + kRows * D + row);
                        const float f = pm == -INFINITY ? 0.f : ex2(pm - m);
                        const float2 a = __ldcg(reinterpret_cast<const float2*>(part + row * D + d));
                        v.x = fmaf(f, a.x, v.x); v.y = fmaf(f, a.y, v.y);
                        l = fmaf(f, __ldcg(part + kRows * D + kRows + row), l);
                    }
                    store(row, d, v, l);
                }
            }
        }
        __syncthreads();                                                // the merge buffer becomes the ring again
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        u = seg0 + blk1;
    }
}

template <typename T, int D, int GS, int NT>
int launch_attn_t(const AttnParams& P, int sms, cudaStream_t stream) {
    using C = AttnCfg<D, GS, NT>;
    static bool attr_done[64] = {};
    int dev = 0;
    CB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        CB_CUDA_TRY(cudaFuncSetAttribute(kv4_attention_kernel<T, D, GS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    kv4_attention_kernel<T, D, GS, NT><<<sms * C::kCtasPerSm, kThreads, C::kSmem, stream>>>(P);
    CB_CUDA_TRY(cudaGetLastError());
    return CB_OK;
}

}  // namespace

// Query rows of a tile: 8, or 16 where a key head has more than 8.
static int attn_tile_rows(int64_t rows) { return rows > 8 ? 16 : 8; }

int64_t kv4_attention_segments(int64_t B, int64_t rows, int64_t kv_heads) {
    const int64_t tile = attn_tile_rows(rows);
    return B * kv_heads * ((rows + tile - 1) / tile);
}

size_t kv4_attention_partial_bytes(int64_t rows, int head_dim) {
    const int sms = sm_count_current();
    if (sms <= 0) return 0;
    const int tile = attn_tile_rows(rows);
    return (size_t)sms * (tile == 8 ? 2 : 1) * 2 * tile * (head_dim + 2) * sizeof(float);
}

// Arguments are checked by the caller.
int launch_kv4_attention(const cb_kv4_cache* c, const void* q, const int64_t* q_strides, void* out, int64_t B, int64_t T, int64_t H,
                         const int32_t* table, int64_t table_stride, const int32_t* lengths, float scale, int* counters,
                         float* partial, cudaStream_t stream) {
    AttnParams P{};
    P.c = Kv4View{reinterpret_cast<unsigned char*>(c->pages), c->n_pages, (int)c->kv_heads, c->page_size / kKvBlock, table, table_stride};
    P.q = q; P.q_b = q_strides[0]; P.q_t = q_strides[1]; P.q_h = q_strides[2];
    P.out = out; P.lengths = lengths; P.B = B; P.T = (int)T; P.H = (int)H; P.G = (int)(H / c->kv_heads);
    P.R = P.T * P.G;
    const int tile = attn_tile_rows(P.R);
    P.row_tiles = (P.R + tile - 1) / tile;
    P.scale_log2 = scale * 1.4426950408889634f;
    P.counters = counters; P.partial = partial;
    const int sms = sm_count_current();
    if (sms <= 0) return CB_ERR_CUDA;
    const bool bf = c->dtype == CB_BF16;
#define CB_KV4_NT(d, gs, nt) (bf ? launch_attn_t<__nv_bfloat16, d, gs, nt>(P, sms, stream) : launch_attn_t<__half, d, gs, nt>(P, sms, stream))
#define CB_KV4_CASE(d, gs) \
    if (c->head_dim == d && c->group_size == gs) return tile == 8 ? CB_KV4_NT(d, gs, 1) : CB_KV4_NT(d, gs, 2);
    CB_KV4_CASE(64, 32) CB_KV4_CASE(64, 64) CB_KV4_CASE(128, 32) CB_KV4_CASE(128, 64) CB_KV4_CASE(128, 128)
#undef CB_KV4_CASE
#undef CB_KV4_NT
    set_error("kv4_attention: no kernel for head_dim %d, group_size %d", c->head_dim, c->group_size);
    return CB_ERR_UNSUPPORTED;
}

int kv4_attn_status_read_and_clear(int* out) {
    int v = 0, zero = 0;
    CB_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_kv4_attn_status, sizeof(int)));
    CB_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_attn_status, &zero, sizeof(int)));
    *out = v;
    return CB_OK;
}

}  // namespace cb
