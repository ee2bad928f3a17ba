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
// that scale's part lies in [2^6, 2^7) for the largest scale met and then rounded to fp16 (w, relative error 2^-11; below 2^-20
// of the largest weight and scale 2^-31 of them).  p is at most 2^8, so that this fits fp16.  What the rounding takes from w is given back for the
// middle of the codes: sum_t w code + sum_t (p (lo + 7.5 scale) - 7.5 w), so that at most 7.5 steps of a value carry it, 2^-11 * 7.5 steps where the format's
// own rounding is half a step (measured: the error against 64 bits falls from 1.7 to 1.1 times that of the fp16 output's rounding, at 1 to 4 % of the
// time).  All sums, the softmax statistics and the lo part are fp32.
//
// Work: the 16-token blocks of all (sequence, row tile, key head) segments form one line that is cut into equal parts, one for each CTA (one to an
// SM), whatever the lengths are; lengths are read on the device, so a captured launch serves any.  The warps of a CTA take
// pairs of blocks in turn, each with a ring of its own filled by bulk copies (one per block), and keep running maxima, sums and
// outputs of their own; they meet in shared memory at the end of a segment.  Where a segment is cut, its parts leave
// (max, sum, output) in scratch and the CTA that arrives last adds them in order of position: the result does not
// depend on timing.
//
// Measured (D = 128, groups of 64): one sequence of 131071 tokens, 64 heads over 8, in 42.7 us, 3.5 TB/s or 0.55 of a copy's rate; sixteen of them
// in 479, 0.78.  The steady state runs at about 0.83 of that rate (the stages of unpacking, products and softmax share the issue slots of three warps on
// each scheduler, which are half busy; a warp's next instruction waits for the one before most of the rest); the rest is the chain of a launch, 12 us long:
// lengths, schedule, look-ups, first copies, the warps' meeting, the join.  16 sequences of 4000 tokens, 32 key heads of one query head: 84 us, 3.5 TB/s.  Of
// caches that the L2 still holds: 24 sequences of 0 to 8192 tokens, 32 heads over 8, 25.4 us, one of 777, 32 heads, 10.1 us, of which that chain is most.
// At D = 128 and groups of 32 the compiler spills 42 bytes (tiles of 16 rows: 82), elsewhere nothing.
#include <algorithm>
#include <cfloat>

#include "cb_kv4.cuh"

namespace cb {
namespace {

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
    bool aligned;                                     // no CTA's part crosses a segment's end, unless there is too much work for that
    int solo;                                         // segments of up to this many blocks are taken by single warps
    float scale_log2;                                 // |softmax scale| * log2(e), above 0
    float q_sign;                                     // 1, or -1 where the scale is negative, 0 where it is 0
    uint32_t zero;                                    // 0, unknown to the compiler
    uint32_t bpp_mul, bpp_shift;                      // n / blocks_per_page = (n * bpp_mul) >> 32 >> bpp_shift for n < 2^31; bpp_mul 0: one block to a page
    int* counters;                                    // [B * kv_heads * row_tiles], zero between calls
    float* partial;                                   // [grid][2][rows of a tile * (D + 2)]
};

// Where a CTA stands: segment `seg` of sequence b (len tokens, nb blocks, per_seg units a segment; base: the sequence's first unit, seg0: the
// segment's), and its blocks of this CTA.
struct Piece {
    uint32_t u, seg0, base, next;                     // next: where the following piece is looked for
    int per_seg, b, seg, nb, len, blk0, blk1;
};
struct Sched { uint32_t u0, u1, share, extra; };

template <int D, int GS, int NT>
struct AttnCfg {
    using L = KvLayout<D, GS>;
    static constexpr int kRows = 8 * NT;
    static constexpr int kWarps = NT == 1 ? 12 : 8, kThreads = kWarps * 32;       // one CTA to an SM: 168 or 255 registers a thread
    static constexpr int kSlotBytes = kStageBlocks * L::kBytes;
    static constexpr int kMerge = kWarps * kRows * D * 4;             // the warps' outputs; then the weights of a cut segment's parts
    // the ring fills what an SM has left; the slots of a warp are at most 8
    static constexpr int kRingBudget = 223 * 1024 - kMerge;
    static constexpr int kSlots = kRingBudget / (kWarps * kSlotBytes) > 8 ? 8 : kRingBudget / (kWarps * kSlotBytes);
    static_assert(kSlots >= 1, "a ring has a slot");
    static constexpr int kMergeOff = kWarps * kSlots * kSlotBytes;
    static constexpr int kStatsOff = kMergeOff + kMerge;              // [2][kWarps][kRows] floats: max, sum
    static constexpr int kBarOff = kStatsOff + 2 * kWarps * kRows * 4;
    static constexpr int kOkOff = kBarOff + kWarps * kSlots * 8;      // [kWarps][kSlots] blocks whose page is good
    static constexpr int kMiscOff = kOkOff + kWarps * kSlots * 4;
    static constexpr int kPlaceOff = kMiscOff + 16, kSchedOff = kPlaceOff + kWarps * 2 * (int)sizeof(Piece);
    static constexpr int kSmem = kSchedOff + kWarps * (int)sizeof(Sched);
    static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
    static constexpr int kPartFloats = kRows * (D + 2);
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    long long t0 = 0;
    for (bool again = false;; again = true) {
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (!again) t0 = clock64();
        else if (clock64() - t0 > kWaitCycles) return false;
    }
}
// A word of 8 codes -> four fp16 pairs: codes 0 and 4 (times 2^-24), 1 and 5 (2^-20), 2 and 6 (2^-24), 3 and 7 (2^-20).  The last
// pair is formed by a subtraction of the two before it, which is exact and runs beside the integer pipe, the busiest one here.
__device__ __forceinline__ void spread(uint32_t w, uint32_t (&a)[4]) {
    a[0] = w & 0x000F000Fu;
    a[1] = w & 0x00F000F0u;
    const uint32_t y = __byte_perm(w, 0u, 0x4341);                // bytes 1 and 3
    a[2] = y & 0x000F000Fu;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&y), *reinterpret_cast<const __half2*>(&a[2]));
    a[3] = *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
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
// Larger of each half; NaN loses.
template <typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max2<__half>(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t max2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <int N> __device__ __forceinline__ void lds_words(const unsigned char* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

__device__ __forceinline__ int arrive(int* counter) {
    int before;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}
// Cached tokens and blocks of a sequence.  The caller has checked that the table's capacity in blocks, times the segments
// of a sequence, fits 31 bits.
__device__ __forceinline__ int seq_len(const AttnParams& P, int64_t b) {
    const int64_t cap = P.c.table_stride * P.c.blocks_per_page * kKvBlock;
    return (int)min((int64_t)max(P.lengths[b], 0), cap);
}
__device__ __forceinline__ int blocks_of(int len) { return (int)(((unsigned)len + kKvBlock - 1) / kKvBlock); }

// How far a score may lie above the reference (in powers of two) before that is moved: p stays below 2^8.
constexpr float kLag = 8.f;

// A weight is 2^(x qmul - m) by one fused operation, and the rounding of the reference m is a factor that all weights of a row share.  It is at most
// 2^0.5 up to m = 2^24; beyond, it would carry p out of fp16's range and then out of a float's.  A warp that has met such an m goes through its blocks
// again, from the references that it has found, halved with their qmul until they are no larger: scores are then held to a step of 1 where they have a
// step of 1 or more in fp32 anyway.
constexpr float kLargeScore = 16777216.f;

// What a segment costs besides its blocks (query rows, the warps' meeting, the join), in blocks.  With 8, 32, 48, 64 and 96 of them: 32 sequences of up to
// 4000 tokens, 32 key heads, take 177, 115, 96, 86 and 89 us; 24 of up to 8192, 8 key heads, 48, 29, 28, 30 and 32; 12 short ones with 12 heads
// 36, 19.9, 18.1, 18.3 and 18.3; 8 of 4000 with 32 rows to a key head 40.8, 40.5, 39.8, 40.5 and 39.5; 32 of 4000 at D = 64 and groups of 32
// 36.5, 36.2, 36.0, 35.4 and 35.4.
constexpr int kOpen = 64;

// Blocks of a CTA up to which parts end with their segment although a tenth of the CTAs or more may then be idle.
constexpr uint32_t kAlignedBlocks = 16;

template <typename T, int D, int GS, int NT>
__global__ void __launch_bounds__((AttnCfg<D, GS, NT>::kThreads), 1)
kv4_attention_kernel(const AttnParams P) {
    using C = AttnCfg<D, GS, NT>;
    using L = typename C::L;
    constexpr int NG = L::NG, kSlots = C::kSlots, kRows = C::kRows, kWarps = C::kWarps, kThreads = C::kThreads;
    constexpr int KW = D / 32, KWG = GS / 32;          // code words of a lane and key row, of one group
    extern __shared__ __align__(128) unsigned char smem[];
    float* merge = reinterpret_cast<float*>(smem + C::kMergeOff);
    float* st_max = reinterpret_cast<float*>(smem + C::kStatsOff);
    float* st_sum = st_max + kWarps * kRows;
    volatile int* misc = reinterpret_cast<volatile int*>(smem + C::kMiscOff);           // [0] abort, [1] last arrival
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

    // ---- the line's length, every warp for itself.  The caller has checked that units fit 32 bits.
    const int B = (int)P.B, first_len = lane < B ? seq_len(P, lane) : 0;              // of sequence `lane`: all there are with up to 32
    // Units of a sequence's segments and how many of these there are.  aligned: a segment of nb blocks is cut into ceil(nb / quota) parts,
    // one to a CTA (quota such that there are CTAs enough), and u counts parts (before quota is known: blocks).  Otherwise the line is cut
    // into equal parts, in which a segment counts kOpen units more than its blocks, ahead of them: what a CTA spends on a segment besides.
    // Short segments (solo) go to single warps, kWarps of them together as one segment that belongs to the CTA in whose part it begins.
    const int groups = (segs + kWarps - 1) / kWarps;
    int quota = 1;
    auto is_solo = [&](int nblk) { return nblk <= P.solo; };
    auto segs_of = [&](int nblk) { return is_solo(nblk) ? groups : segs; };
    bool aligned = P.aligned;
    auto units_of = [&](int nblk) { return aligned ? (nblk + quota - 1) / quota : nblk == 0 ? 0 : is_solo(nblk) ? kOpen + nblk * kWarps : kOpen + nblk; };
    auto all_units = [&]() {
        uint32_t n = (uint32_t)(units_of(blocks_of(first_len)) * segs_of(blocks_of(first_len)));
        for (int s = lane + 32; s < B; s += 32) { const int m = blocks_of(seq_len(P, s)); n += (uint32_t)(units_of(m) * segs_of(m)); }
        return __reduce_add_sync(0xffffffffu, n);
    };
    uint32_t U = all_units();
    // With few CTAs to a segment those that are left over stay idle: only where that costs little beside the rest (32 segments of 131071 tokens on 148
    // SMs: 4 CTAs each, 145 us, cut into equal parts 129; 32 segments of 777 tokens: 10.1 and 10.7).
    if (aligned && 16 * B * segs > (int)gridDim.x && U > kAlignedBlocks * gridDim.x) {
        aligned = false;
        U = all_units();
    }
    // ---- this CTA's part [u0, u1) of the line (the first `extra` parts have a unit more)
    const uint32_t nc = min(gridDim.x, max(U, 1u)), share = U / nc, extra = U - share * nc;
    auto unit_of_cta = [&](uint32_t c) { return share * c + min(c, extra); };
    const uint32_t spare = gridDim.x - (uint32_t)(B * segs);                          // aligned: CTAs beyond one for each segment
    if (aligned) quota = (int)((U + spare - 1u) / spare);
    const uint32_t u0 = aligned ? blockIdx.x : unit_of_cta(blockIdx.x);
    const uint32_t u1 = aligned ? u0 + 1u : unit_of_cta(blockIdx.x + 1u);

    // ---- the sequence that holds unit u0
    int b = -1, len = 0, nb = 0, per_seg = 0;
    uint32_t base = 0;
    if (blockIdx.x < nc || aligned)
        for (int b0 = 0; b0 < B; b0 += 32) {
            const int my_len = b0 == 0 ? first_len : b0 + lane < B ? seq_len(P, b0 + lane) : 0;
            const uint32_t units = (uint32_t)(units_of(blocks_of(my_len)) * segs_of(blocks_of(my_len)));
            uint32_t cum = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, cum, o);
                if (lane >= o) cum += up;
            }
            const unsigned past = __ballot_sync(0xffffffffu, base + cum > u0);
            if (past != 0u) {
                const int l = __ffs(past) - 1;
                b = b0 + l;
                len = __shfl_sync(0xffffffffu, my_len, l);
                base += __shfl_sync(0xffffffffu, cum - units, l);
                break;
            }
            base += __shfl_sync(0xffffffffu, cum, 31);
        }
    // sequences without keys: their rows are zero
    auto zero_rows = [&]() {
        for (int s = blockIdx.x; s < B; s += gridDim.x)
            if (seq_len(P, s) == 0) {
                uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(P.out) + (int64_t)s * P.T * P.H * D);
                for (int i = tid; i < P.T * P.H * D / 2; i += kThreads) o[i] = 0u;
            }
    };
    if (U == 0u || b < 0) { zero_rows(); return; }     // nothing to do, or (aligned) more CTAs than parts
    nb = blocks_of(len);
    per_seg = units_of(nb);

    // ---- a piece: the blocks [blk0, blk1) of one segment.  Where the CTA stands in its list is needed between pieces only: it waits in
    // shared memory (every warp has its own), the registers are for the product.
    Piece* place = reinterpret_cast<Piece*>(smem + C::kPlaceOff) + warp * 2;
    Sched* sched = reinterpret_cast<Sched*>(smem + C::kSchedOff) + warp;
    // The piece that begins at unit `at` or behind it, before `end`; false where there is none.  p: a sequence, `at` not before it.
    auto piece_at = [&](Piece& p, uint32_t at, uint32_t end) {
        for (;;) {
            while (at >= p.base + (uint32_t)(p.per_seg * segs_of(p.nb))) {
                p.base += (uint32_t)(p.per_seg * segs_of(p.nb));
                if (++p.b >= B) return false;
                p.len = seq_len(P, p.b);
                p.nb = blocks_of(p.len);
                p.per_seg = units_of(p.nb);
            }
            if (at >= end) return false;
            const uint32_t local = at - p.base;
            p.u = at;
            p.seg = (int)(local / (uint32_t)p.per_seg);
            const int part = (int)(local - (uint32_t)p.seg * (uint32_t)p.per_seg);
            p.seg0 = at - (uint32_t)part;
            p.next = p.seg0 + (uint32_t)p.per_seg;
            if (aligned) {
                const int each = p.nb / p.per_seg, more = p.nb - each * p.per_seg;
                p.blk0 = each * part + min(part, more);
                p.blk1 = p.blk0 + each + (part < more ? 1 : 0);
                p.next = end;
                return true;
            }
            if (is_solo(p.nb)) {
                p.blk0 = 0; p.blk1 = p.nb;
                if (part == 0) return true;
                at = p.next;                           // begun, and finished, by an earlier CTA
                continue;
            }
            p.blk0 = max(part - kOpen, 0);
            p.blk1 = min(p.nb, (int)(end - p.seg0) - kOpen);
            return p.blk1 > p.blk0;                    // else nothing but the opening
        }
    };
    int b_now, seg_now, len_now, blk0, blk1;
    bool solo;                                         // this warp has the segment to itself
    auto enter = [&](const Piece& p) {
        solo = !aligned && is_solo(p.nb);
        b_now = p.b; len_now = p.len; blk0 = p.blk0; blk1 = p.blk1;
        seg_now = p.seg;
        if (solo) {
            seg_now = p.seg * kWarps + warp;
            if (seg_now >= segs) { seg_now = 0; blk1 = 0; }            // nothing for this warp
        }
    };
    {
        Piece p;
        p.base = base; p.b = b; p.len = len; p.nb = blocks_of(len); p.per_seg = units_of(p.nb);
        if (!piece_at(p, u0, u1)) { zero_rows(); return; }
        enter(p);
        if (lane == 0) { place[0] = p; *sched = Sched{u0, u1, share, extra}; }
    }

    // ---- this warp's stages of the piece: stage i holds `per` blocks from first(i) on; few blocks: one to a stage
    uint32_t it = 0;                                   // stages this warp has taken from its ring, ever
    int per = 1, mine = 0;
    const int32_t* table_row = nullptr;
    const unsigned char* head_pages = nullptr;
    auto first_of = [&](int i) { return blk0 + (solo ? i : warp + i * kWarps) * per; };
    auto page_of = [&](int blk, int& in_page) {        // of a block of this piece, or -1
        const int row = P.bpp_mul == 0u ? blk : (int)(__umulhi((uint32_t)blk, P.bpp_mul) >> P.bpp_shift);
        in_page = blk - row * P.c.blocks_per_page;
        const int page = table_row[row];
        if (page >= 0 && page < P.c.n_pages) return page;
        atomicExch(&g_kv4_attn_status, kKv4BadPage);
        return -1;
    };
    auto expect = [&](uint32_t s, unsigned good) {     // one lane
        slot_ok[s] = good;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bars + 8 * s), "r"((uint32_t)(__popc(good) * L::kBytes)) : "memory");
    };
    auto copy = [&](uint32_t s, int c, int page, int in_page) {
        const unsigned char* src = head_pages + ((int64_t)page * kv_heads * P.c.blocks_per_page + in_page) * L::kBytes;
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(ring_u32 + s * C::kSlotBytes + c * L::kBytes), "l"(src), "r"((uint32_t)L::kBytes), "r"(bars + 8 * s) : "memory");
    };
    auto issue = [&](int i, uint32_t at) {
        const uint32_t s = at % kSlots;
        const int blk = first_of(i) + lane;
        int page = -1, in_page = 0;
        if (lane < per && blk < blk1) page = page_of(blk, in_page);
        const unsigned good = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) expect(s, good);
        __syncwarp();
        if (page >= 0) copy(s, lane, page, in_page);
    };
    // The first stages of a piece: lane 2 i + c brings block c of stage i, so that all look-ups wait for memory together (one after another they took 3 us).
    static_assert(kSlots * kStageBlocks <= 32, "a lane for each block of the ring");
    auto issue_first = [&]() {
        const int i = lane / kStageBlocks, c = lane % kStageBlocks, blk = first_of(i) + c;
        const uint32_t s = (it + i) % kSlots;
        const bool some = i < kSlots && i < mine;
        int page = -1, in_page = 0;
        if (some && c < per && blk < blk1) page = page_of(blk, in_page);
        const unsigned good = __ballot_sync(0xffffffffu, page >= 0);
        if (some && c == 0) expect(s, (good >> lane) & ((1u << kStageBlocks) - 1u));
        __syncwarp();
        if (page >= 0) copy(s, c, page, in_page);
    };
    auto begin_piece = [&](int b, int seg) {           // the first stages of a piece are on their way before anything else
        const int pieces = blk1 - blk0;
        per = solo || pieces > 2 * kWarps ? kStageBlocks : 1;
        const int nstage = (pieces + per - 1) / per;
        mine = solo ? nstage : warp < nstage ? (nstage - 1 - warp) / kWarps + 1 : 0;
        table_row = P.c.table + (int64_t)b * P.c.table_stride;
        head_pages = P.c.pages + (int64_t)(seg % kv_heads) * P.c.blocks_per_page * L::kBytes;
        issue_first();
    };
    __syncthreads();                                   // barriers are there
    begin_piece(b_now, seg_now);
    zero_rows();

    bool again = false;                                // this warp's second time through the piece
    for (int bank = 0;; bank ^= 1) {
        const int row0 = seg_now / kv_heads * kRows, len = len_now;

        // ---- query rows: fp16 fragments, their scales, sums and limits
        uint32_t qf[NT][KW * 4];
        float qsum[NT][NG][2], qmul[NT][2];
        int lim[NT][2], seen_by_all = 0x7fffffff;            // the smallest limit of the tile's rows; those behind the last (q = 0, not stored) have none
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row0 + n * 8 + g;
            const bool live = r < P.R;
            const int rt = live ? r / P.G : 0, rg = live ? r % P.G : 0;
            const T* src = reinterpret_cast<const T*>(P.q) + (int64_t)b_now * P.q_b + rt * P.q_t + (int64_t)(seg_now % kv_heads * P.G + rg) * P.q_h;
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
            // 2^(140 - e).  With an infinity among a row's values each score is an infinity or NaN, and none above -inf if they are infinities of one
            // sign: no softmax survives that, so the row's values become NaN at once, and its sum with them.
            const float f = mx < INFINITY ? P.q_sign * __uint_as_float((uint32_t)(267 - e) << 23) : __int_as_float(0x7fffffff);
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
            // Kept among the normal floats: 0 times the -inf of an unseen token, or an infinity times a score, would be NaN.  Where that changes it, the row's
            // values are all below 2^-112 (the scores are then 0 in effect) or above 2^119 (one key has all the weight).
            const float mul = fminf(fmaxf(P.scale_log2 * 16777216.f * __uint_as_float((uint32_t)(e - 13) << 23), FLT_MIN), FLT_MAX);
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
                if (row0 + n * 8 + 2 * t + c < P.R) seen_by_all = min(seen_by_all, lim[n][c]);
            }
        }
        const int plain_end = max(__reduce_min_sync(0xffffffffu, seen_by_all), 0) / kKvBlock;      // blocks before it are seen whole by every row

        float o[NT][D / 16][4], m_run[NT][2], l_run[NT][2], z[NT][NG][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m_run[n][c] = -INFINITY; l_run[n][c] = 0.f;
                if (again)
                    for (m_run[n][c] = st_max[warp * kRows + n * 8 + 2 * t + c]; fabsf(m_run[n][c]) > kLargeScore && fabsf(m_run[n][c]) < INFINITY; m_run[n][c] *= 0.5f) qmul[n][c] *= 0.5f;
#pragma unroll
                for (int j = 0; j < NG; ++j) z[n][j][c] = 0.f;
            }
        }
        int s_exp = 15;                                // exponent field of the power of two that p * scale is divided by

        const int ra = g & 1 ? 7 - (g >> 1) : (g >> 1);            // token of accumulator row g; row g + 8 is token ra + 8
        const int va_off = L::kVCodes + t * D + L::v_piece(g, t);  // this lane's piece of token pair t; pair t + 4 is 4 D further

        // One stage: scores, running maxima, weights, weighted values.  PLAIN: both blocks there, every token seen by every row.
        auto take = [&](auto plain_tag, const unsigned char* stage, int first, unsigned good) -> uint32_t {
            constexpr bool PLAIN = decltype(plain_tag)::value;
            float x[kStageBlocks][NT][4];
            uint32_t smax2 = 0u;                                   // largest (scale, lo) of the values, as a pair; only scale is used
#pragma unroll
            for (int k = 0; k < kStageBlocks; ++k) {
                if (!PLAIN && !((good >> k) & 1u)) {
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
                float acc[NG][NT][4];
#pragma unroll
                for (int wg = 0; wg < KWG; ++wg)
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        const int w = j * KWG + wg;
                        uint32_t a[4], c[4];
                        spread(wa[w], a);
                        spread(wb[w], c);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (wg == 0) mma16816_first(acc[j][n], a[0], c[0], a[1], c[1], qf[n][4 * w], qf[n][4 * w + 1]);
                            else mma16816(acc[j][n], a[0], c[0], a[1], c[1], qf[n][4 * w], qf[n][4 * w + 1]);
                            mma16816(acc[j][n], a[2], c[2], a[3], c[3], qf[n][4 * w + 2], qf[n][4 * w + 3]);
                        }
                    }
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const float2 sa = unpack2<T>(ma[j]), sb = unpack2<T>(mb[j]);     // (scale, lo)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            x[k][n][c] = fmaf(acc[j][n][c], sa.x, j == 0 ? sa.y * qsum[n][j][c] : fmaf(sa.y, qsum[n][j][c], x[k][n][c]));
                            x[k][n][2 + c] = fmaf(acc[j][n][2 + c], sb.x, j == 0 ? sb.y * qsum[n][j][c] : fmaf(sb.y, qsum[n][j][c], x[k][n][2 + c]));
                        }
                }
                uint32_t va[NG], vb[NG];
                lds_words<NG>(blk + L::kVMeta + ra * L::kMeta, va);
                lds_words<NG>(blk + L::kVMeta + (ra + 8) * L::kMeta, vb);
                const int tok = (first + k) * kKvBlock + ra;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    smax2 = max2<T>(smax2, PLAIN || tok < len ? va[j] : 0u);
                    smax2 = max2<T>(smax2, PLAIN || tok + 8 < len ? vb[j] : 0u);
                }
                if constexpr (!PLAIN) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (tok >= lim[n][c]) x[k][n][c] = -INFINITY;
                            if (tok + 8 >= lim[n][c]) x[k][n][2 + c] = -INFINITY;
                        }
                }
            }
            // ---- m_run follows the running maximum of the scaled scores, s_exp that of the value scales.  m_run is moved only where
            // some score lies more than kLag above it: p stays below 2^kLag, and most stages need no exchange between lanes.
            const float smax = fmaxf(unpack2<T>(smax2).x, 0.f);
            float mx[NT][2];
            bool move = (int)(__float_as_uint(smax) >> 23) > s_exp;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(x[0][n][c], x[0][n][2 + c]);
#pragma unroll
                    for (int k = 1; k < kStageBlocks; ++k) m = fmaxf(m, fmaxf(x[k][n][c], x[k][n][2 + c]));
                    mx[n][c] = m * qmul[n][c];
                    move = move || mx[n][c] > m_run[n][c] + kLag;
                }
            if (__any_sync(0xffffffffu, move)) {
                const int e_new = max(s_exp, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(smax)) >> 23));
                const float rs = __uint_as_float((uint32_t)max(127 + s_exp - e_new, 0) << 23);
                s_exp = e_new;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float alpha[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float m = mx[n][c];
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                        m = fmaxf(m_run[n][c], m);
                        alpha[c] = m == m_run[n][c] ? 1.f : ex2(m_run[n][c] - m);
                        m_run[n][c] = m;
                        l_run[n][c] *= alpha[c];
#pragma unroll
                        for (int j = 0; j < NG; ++j) z[n][j][c] *= alpha[c];
                        alpha[c] *= rs;
                    }
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        o[n][d][0] *= alpha[0]; o[n][d][1] *= alpha[1];
                        o[n][d][2] *= alpha[0]; o[n][d][3] *= alpha[1];
                    }
                }
            }
            const float cmul = __uint_as_float((uint32_t)(260 - s_exp) << 23);       // 2^6 / 2^(s_exp - 127)
            const float centre = -7.5f * __uint_as_float((uint32_t)(s_exp - 6) << 23);      // -7.5 / cmul
            uint32_t words = 0u;
#pragma unroll
            for (int k = 0; k < kStageBlocks; ++k) {
                if (!PLAIN && !((good >> k) & 1u)) continue;
                const unsigned char* blk = stage + k * L::kBytes;
                uint32_t va[NG], vb[NG];
                lds_words<NG>(blk + L::kVMeta + ra * L::kMeta, va);
                lds_words<NG>(blk + L::kVMeta + (ra + 8) * L::kMeta, vb);
                float p[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float m = !PLAIN && m_run[n][c] == -INFINITY ? 0.f : m_run[n][c];
                        p[n][c] = ex2(fmaf(x[k][n][c], qmul[n][c], -m));
                        p[n][2 + c] = ex2(fmaf(x[k][n][2 + c], qmul[n][c], -m));
                        l_run[n][c] += p[n][c] + p[n][2 + c];
                    }
                uint32_t pb[NT][NG][2];
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const float2 sa = unpack2<T>(va[j]), sb = unpack2<T>(vb[j]);
                    const float fa = sa.x * cmul, fb = sb.x * cmul;
                    const float mid_a = fmaf(7.5f, sa.x, sa.y), mid_b = fmaf(7.5f, sb.x, sb.y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if constexpr (PLAIN) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) z[n][j][c] = fmaf(p[n][c], mid_a, fmaf(p[n][2 + c], mid_b, z[n][j][c]));
                            const uint32_t wa = pack_h2(p[n][0] * fa, p[n][1] * fa), wb = pack_h2(p[n][2] * fb, p[n][3] * fb);
                            const float2 ga = unpack2<__half>(wa), gb = unpack2<__half>(wb);
                            z[n][j][0] = fmaf(ga.x, centre, fmaf(gb.x, centre, z[n][j][0]));
                            z[n][j][1] = fmaf(ga.y, centre, fmaf(gb.y, centre, z[n][j][1]));
                            pb[n][j][0] = movmatrix_t(wa);
                            pb[n][j][1] = movmatrix_t(wb);
                        } else {
                            // what a row does not see adds nothing, whatever is stored there; what it sees with a weight too small for a float does
                            float h[4] = {p[n][0] * fa, p[n][1] * fa, p[n][2] * fb, p[n][3] * fb};
                            float y[4] = {p[n][0] * mid_a, p[n][1] * mid_a, p[n][2] * mid_b, p[n][3] * mid_b};
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (x[k][n][c] == -INFINITY) h[c] = y[c] = 0.f;
                            const uint32_t wa = pack_h2(h[0], h[1]), wb = pack_h2(h[2], h[3]);
                            const float2 ga = unpack2<__half>(wa), gb = unpack2<__half>(wb);
                            z[n][j][0] += fmaf(ga.x, centre, y[0]) + fmaf(gb.x, centre, y[2]);
                            z[n][j][1] += fmaf(ga.y, centre, y[1]) + fmaf(gb.y, centre, y[3]);
                            pb[n][j][0] = movmatrix_t(wa);
                            pb[n][j][1] = movmatrix_t(wb);
                        }
                    }
                }
                uint32_t v0[D / 32], v1[D / 32];                                     // pairs t and t + 4
                lds_words<D / 32>(blk + va_off, v0);
                lds_words<D / 32>(blk + va_off + 4 * D, v1);
#pragma unroll
                for (int hw = 0; hw < D / 32; ++hw) {                                // four values of this lane, two tokens each
                    const int j = hw * 4 / (GS / 8);
                    uint32_t a[4], c[4];
                    spread(v0[hw], a);
                    spread(v1[hw], c);
                    words |= v0[hw] | v1[hw];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816(o[n][2 * hw], a[0], a[2], c[0], c[2], pb[n][j][0], pb[n][j][1]);
                        mma16816(o[n][2 * hw + 1], a[1], a[3], c[1], c[3], pb[n][j][0], pb[n][j][1]);
                    }
                }
            }
            return words;
        };

        for (int i = 0; i < mine; ++i) {
            const uint32_t at = it + i, s = at % kSlots;
            if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * s, (at / kSlots) & 1))) {
                if (lane == 0) { misc[0] = 1; atomicExch(&g_kv4_attn_status, kKv4Wait); }
                for (int k = i + 1; k < mine && k < i + kSlots; ++k) mbar_wait(bars + 8 * ((it + k) % kSlots), ((it + k) / kSlots) & 1);
                break;
            }
            const int first = first_of(i);
            const unsigned good = slot_ok[s];
            const unsigned char* stage = ring + s * C::kSlotBytes;
            const int cnt = min(per, blk1 - first);
            // A stage of whole blocks that every row sees needs no masks (16 sequences of 4000 tokens, 32 key heads of one query head: 84 us, with masks 95).
            uint32_t seen_words;
            if (good == 3u && cnt == kStageBlocks && first + cnt <= plain_end) seen_words = take(std::true_type{}, stage, first, good);
            else seen_words = take(std::false_type{}, stage, first, good);
            // The slot may be overwritten once every lane has its codes in registers: this vote needs the V words (masked with a zero
            // that the compiler does not know), the vote on the maxima needed all else.
            const unsigned held = __ballot_sync(0xffffffffu, (seen_words & P.zero) != 0u);
            if (i + kSlots < mine) issue(i + kSlots, at + kSlots + held);
        }
        it += mine;
        bool large = false;                            // a reference is, or was, beyond kLargeScore
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                large = large || (fabsf(m_run[n][c]) > kLargeScore && fabsf(m_run[n][c]) < INFINITY) || !(fabsf(l_run[n][c] + z[n][0][c]) < INFINITY);
        const bool redo = __any_sync(0xffffffffu, large) && !again;

        // ---- the next piece's copies start, or this one's again
        const bool alone = solo, idle = solo && blk1 == 0, whole = blk0 == 0 && blk1 == place[bank].nb;
        const int64_t first_row = (int64_t)b_now * P.T * P.H + seg_now % kv_heads * P.G;      // of the output, in rows of D: row r is T's r / G, head r % G
        bool begun = false;
        if (misc[0] == 0) {
            Piece p = place[bank];
            if (redo || piece_at(p, p.next, sched->u1)) {
                if (!redo) {
                    enter(p);
                    if (lane == 0) place[bank ^ 1] = p;
                }
                begin_piece(b_now, seg_now);
                begun = true;
            }
        }
        if (redo && begun) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) st_max[warp * kRows + n * 8 + 2 * t + c] = m_run[n][c];      // the same from every g
            again = true;
            bank ^= 1;
            continue;
        }

        // ---- the warps' results meet: value = o * 2^24 (2^20) / cmul + z
        {
            const float back = __uint_as_float((uint32_t)(s_exp - 6) << 23);         // 1 / cmul
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
                    if (g == 0) {
                        if (!again) st_max[warp * kRows + row] = m_run[n][c];           // the second time it stands there, before any halving
                        st_sum[warp * kRows + row] = l;
                    }
                    float* dst = merge + ((size_t)warp * kRows + row) * D;
#pragma unroll
                    for (int hw = 0; hw < D / 32; ++hw) {
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
        again = false;
        if (!alone) __syncthreads(); else __syncwarp();
        if (misc[0] != 0) {                                             // a copy was not heard of: wait (bounded) for the others in flight
            if (begun)
                for (int i = 0; i < kSlots && i < mine; ++i) mbar_wait(bars + 8 * ((it + i) % kSlots), ((it + i) / kSlots) & 1);
            return;
        }
        const Piece& now = place[bank];
        auto store = [&](int row, int d, auto& v, float l) {            // neighbouring values of a finished row
            constexpr int N = sizeof(v) / sizeof(float);
            const int r = row0 + row;
            if (r >= P.R) return;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            T y[N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = from_f32<T>(l == 0.f ? 0.f : v[i] * inv);
            T* dst = reinterpret_cast<T*>(P.out) + (first_row + (int64_t)(r / P.G) * P.H + r % P.G) * D + d;
            if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
            else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(y);
        };
        if (alone) {                                                    // this warp's rows are finished
            if (!idle)
                for (int idx = lane; idx < kRows * D / 4; idx += 32) {
                    const int row = idx / (D / 4), d = idx % (D / 4) * 4;
                    const float4 a = *reinterpret_cast<const float4*>(merge + ((size_t)warp * kRows + row) * D + d);
                    float v[4] = {a.x, a.y, a.z, a.w};
                    store(row, d, v, st_sum[warp * kRows + row]);
                }
            if (!begun) return;
            __syncwarp();
            continue;
        }
        float* my_part = P.partial + ((int64_t)blockIdx.x * 2 + (now.u == sched->u0 ? 0 : 1)) * C::kPartFloats;
        for (int idx = tid; idx < kRows * D / 4; idx += kThreads) {
            const int row = idx / (D / 4), d = idx % (D / 4) * 4;
            float mw[kWarps], m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) { mw[w] = st_max[w * kRows + row]; m = fmaxf(m, mw[w]); }
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float sw = st_sum[w * kRows + row];
                if (mw[w] == -INFINITY && sw == 0.f) continue;          // saw nothing; where all scores are NaN the sum is NaN, and stays
                const float f = ex2(mw[w] - m);
                const float4 a = *reinterpret_cast<const float4*>(merge + ((size_t)w * kRows + row) * D + d);
                v[0] = fmaf(f, a.x, v[0]); v[1] = fmaf(f, a.y, v[1]); v[2] = fmaf(f, a.z, v[2]); v[3] = fmaf(f, a.w, v[3]);
                l = fmaf(f, sw, l);
            }
            if (whole) store(row, d, v, l);
            else {
                *reinterpret_cast<float4*>(my_part + row * D + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) { my_part[kRows * D + row] = m; my_part[kRows * D + kRows + row] = l; }
            }
        }
        if (!whole) {
            // CTAs that hold the segment's first and last block: c0 .. c0 + n - 1
            const uint32_t share = sched->share, extra = sched->extra;
            auto cta_of_unit = [&](uint32_t u) { return u < extra * (share + 1u) ? u / (share + 1u) : extra + (u - extra * (share + 1u)) / share; };
            const uint32_t c0 = aligned ? now.seg0 : cta_of_unit(now.seg0 + kOpen);
            const int n = aligned ? now.per_seg : (int)(cta_of_unit(now.seg0 + (uint32_t)now.per_seg - 1u) - c0) + 1;
            __syncthreads();
            if (tid == 0) {
                int* counter = P.counters + ((int64_t)now.b * segs + now.seg);
                // the CTA's part, ordered before by the barrier, is visible to who sees the count, and the others' to this CTA if it is the last
                const bool last = arrive(counter) == n - 1;
                if (last) *counter = 0;
                misc[1] = last;
            }
            __syncthreads();
            if (misc[1] != 0) {
                // Parts lie at c0 (its second one, if the segment does not begin with that CTA), c0 + 1, ...  A warp takes a row, a lane
                // 4 values of it (2 at D = 64).
                const int64_t off0 = ((int64_t)c0 * 2 + (aligned || share * c0 + min(c0, extra) >= now.seg0 ? 0 : 1)) * C::kPartFloats;
                auto part = [&](int c) { return P.partial + (c == 0 ? off0 : (int64_t)(c0 + c) * 2 * C::kPartFloats); };
                constexpr int kV = D / 32;
                for (int row = warp; row < kRows; row += kWarps) {
                    float* weight = merge + row * n;
                    // a part's maximum and sum for each lane (further ones where there are more than 32), and the first outputs, on their way together
                    constexpr int kAhead = 8;
                    float pm = lane < n ? __ldcg(part(lane) + kRows * D + row) : -INFINITY, pl = lane < n ? __ldcg(part(lane) + kRows * D + kRows + row) : 0.f;
                    float a[kAhead][kV];
                    auto fetch = [&](int c) {
#pragma unroll
                        for (int k = 0; k < kAhead; ++k)
                            if (c + k < n) {
                                const float* src = part(c + k) + row * D + lane * kV;
                                if constexpr (kV == 4) {
                                    const float4 q4 = __ldcg(reinterpret_cast<const float4*>(src));
                                    a[k][0] = q4.x; a[k][1] = q4.y; a[k][2] = q4.z; a[k][3] = q4.w;
                                } else {
                                    const float2 q2 = __ldcg(reinterpret_cast<const float2*>(src));
                                    a[k][0] = q2.x; a[k][1] = q2.y;
                                }
                            }
                    };
                    fetch(0);
                    float m = pm, l = 0.f;
                    for (int c = lane + 32; c < n; c += 32) m = fmaxf(m, __ldcg(part(c) + kRows * D + row));
#pragma unroll
                    for (int o2 = 16; o2 > 0; o2 >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
                    for (int c = lane; c < n; c += 32) {
                        if (c >= 32) { pm = __ldcg(part(c) + kRows * D + row); pl = __ldcg(part(c) + kRows * D + kRows + row); }
                        const float f = pm == -INFINITY && pl == 0.f ? 0.f : ex2(pm - m);     // nothing seen: 0; NaN stays
                        weight[c] = f;
                        l = fmaf(f, pl, l);
                    }
#pragma unroll
                    for (int o2 = 16; o2 > 0; o2 >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o2);
                    __syncwarp();
                    float v[kV];
#pragma unroll
                    for (int i = 0; i < kV; ++i) v[i] = 0.f;
                    for (int c = 0;;) {
#pragma unroll
                        for (int k = 0; k < kAhead; ++k)
                            if (c + k < n) {
                                const float f = weight[c + k];
#pragma unroll
                                for (int i = 0; i < kV; ++i) v[i] = fmaf(f, a[k][i], v[i]);
                            }
                        if ((c += kAhead) >= n) break;
                        fetch(c);
                    }
                    store(row, lane * kV, v, l);
                }
            }
        }
        if (!begun) return;
        __syncthreads();                                                // merge, st_max and st_sum are free again
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
    // a cut segment has at most one part on each CTA: their weights share the merge buffer
    if (sms > C::kWarps * D) { set_error("kv4_attention: more SMs than this kernel was laid out for"); return CB_ERR_UNSUPPORTED; }
    kv4_attention_kernel<T, D, GS, NT><<<sms, C::kThreads, C::kSmem, stream>>>(P);
    CB_CUDA_TRY(cudaGetLastError());
    return CB_OK;
}

}  // namespace

// Query rows of a tile: 8, or 16 where a key head has more than 8.  (4 rows in tiles of 16: 37.9 us for 30.0, 8 rows 63.9 for 42.2.)
static int attn_tile_rows(int64_t rows) { return rows > 8 ? 16 : 8; }

int64_t kv4_attention_segments(int64_t B, int64_t rows, int64_t kv_heads) {
    const int64_t tile = attn_tile_rows(rows);
    return B * kv_heads * ((rows + tile - 1) / tile);
}

size_t kv4_attention_partial_bytes(int64_t rows, int head_dim) {
    const int sms = sm_count_current();
    if (sms <= 0) return 0;
    const int tile = attn_tile_rows(rows);
    return (size_t)sms * 2 * tile * (head_dim + 2) * sizeof(float);
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
    P.q_sign = scale < 0.f ? -1.f : scale > 0.f ? 1.f : 0.f;
    P.scale_log2 = scale == 0.f ? 1.f : std::min(fabsf(scale) * 1.4426950408889634f, FLT_MAX);         // a scale of 0 weighs all keys alike: queries of 0 do
    P.zero = 0u;
    {   // with 2^s >= d > 2^(s - 1), m = ceil(2^(31 + s) / d) < 2^32 is off by less than 1, n * m / 2^(31 + s) by less than n / 2^(31 + s) < 1 / d
        const uint32_t d = (uint32_t)P.c.blocks_per_page;
        uint32_t s = 0;
        while ((1u << s) < d) ++s;
        P.bpp_mul = d == 1u ? 0u : (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
        P.bpp_shift = d == 1u ? 0u : s - 1;
    }
    P.counters = counters; P.partial = partial;
    const int sms = sm_count_current();
    if (sms <= 0) return CB_ERR_CUDA;
    // Few segments: parts that end with their segment, so that each CTA goes through the chain of copy, product and join once (8 segments of
    // 131071 tokens: 42.2 us, cut into equal parts 43.4); the parts are then up to a quarter longer.  Many: equal parts.
    P.aligned = 4 * B * c->kv_heads * P.row_tiles <= sms;
    // Segments enough to fill the SMs: the short ones (up to 128 tokens) one to a warp (512 segments of 100 tokens: 13.5 us, by whole CTAs
    // 23.6; where a fifth are that short, 192 segments of up to 8192: 30.0 and 27.5).
    P.solo = !P.aligned && B * c->kv_heads * P.row_tiles >= sms ? 8 : 0;
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
