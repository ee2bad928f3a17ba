// Attention of whole prompts on tcgen05: out_i = sum_{j <= i + Lk - Lq} softmax_j(scale * q_i . k_j) v_j for packed sequences of
// different lengths, grouped heads, with or without the causal bound.
//
// One persistent CTA per SM takes tiles of 256 query rows of one head and sequence, as two sub-tiles of 128 rows, and walks over key
// tiles of 128.  For each sub-tile and key tile
//     S = Q K^T     128 x 128 x D, both operands in shared memory (K-major), fp32 in tensor memory
//     p = exp2(c s - m), l += sum p, m a reference that follows the running maximum
//     O += P V      128 x D x 128, P in 16 bits in tensor memory over S's columns, V as it lies in memory (N-major operand)
// The two sub-tiles alternate: while the softmax warps of one work on its scores, the tensor cores run the other's products.
// A thread of the softmax warps owns a row (a TMEM lane), so maxima and sums need no exchange.  The reference m is moved only
// when the maximum has grown by more than 2^8 (then O and l are rescaled), which makes rescaling rare: p stays below 256, and its 16-bit
// rounding is relative.  p is rounded to the inputs' type, which is what the product with V takes (error of the whole output against 64 bits: bf16 2.0e-3
// where its own rounding is 1.6e-3, fp16 2.2e-4 to 2.5e-4 and 2.0e-4); the sum l takes the unrounded p.
//
// TMEM map (512 columns): S0/P0 [0, 128), S1/P1 [128, 256), O0 [256, 256 + D), O1 [384, 384 + D).
// Warps: 0-3 softmax and epilogue of sub-tile 0, 4-7 of sub-tile 1, 8 TMA, 9 MMA, 10 the walk through
// the work, 11 zeros behind the last key (below).  Warps 8-11 give registers to the softmax warps, which hold a whole row of scores.
//
// What a row does not see gets weight 0, but 0 * inf is not 0.  V rows behind the last key of a sequence belong to another sequence (or to
// nothing) and are zeroed in shared memory.  Inside a sequence, where a value that is not finite follows a row within its last key tiles, the row's
// sum comes out as NaN; the epilogue looks for that (it adds the row up) and forms such a sum again, from memory and without the tensor cores.
// K needs nothing: scores are masked by selection.
//
// What bounds it at D = 128: 4 * 128 * 128 * D operations of a sub-tile and key tile are 1024 clocks of the tensor cores, and
// its 128 * 128 exponentials are 1024 clocks of the special-function units; at D = 64 these are twice the products' time.  So the softmax warps may not
// lose issue slots: packed fp32 arithmetic, a row to a thread, nothing unrolled that runs once a tile.
//   16384 tokens, 32 heads, D = 128, causal, bf16:            1.72 to 1.81 ms in a replayed graph, 1220 to 1280 TFLOP/s; 2.0 ms, 1100 TFLOP/s, in calls that
//                                                              follow one another on new inputs: the GPU is at its power limit, and runs differ by as much
//   12 prompts of 1 to 4096 tokens, 32 heads over 8, D = 128: 262 us (calls: 301), 920 TFLOP/s of what the pairs need; tiles on the diagonal and at
//                                                              prompts' ends, and a tile's opening and epilogue (kOpen), are the rest
//   4 prompts of 4096, 32 heads over 8, D = 128, not causal:  0.89 ms, 1230 TFLOP/s
//   16384 tokens, 16 heads, D = 64, causal, fp16:             840 to 920 us, 600 to 655 TFLOP/s
//   one prompt of 37 tokens, 32 heads:                        10 us (calls: 15): launch, tensor maps, TMEM, one pass through the roles
// The compiler spills 76 to 88 bytes of a softmax thread's registers at 168 a thread at launch.
//
// Every wait is bounded; a wait that runs out raises a flag in shared memory and the status word, every role leaves its
// loops, TMEM is released, and the kernel returns.
#include <algorithm>
#include <cfloat>

#include "cb_common.cuh"
#include "cb_f32x2.cuh"

namespace cb {
namespace {

constexpr int kSub = 128, kTileQ = 2 * kSub, kTileK = 128;
constexpr int kOpen = 3;                              // what a CTA spends on a (tile, head) besides its products, in key tiles (the 12 prompts with 1: 272 us)
// A round is kRoundUnits units for a CTA, or more: 16384 tokens, 32 heads took 1.69 to 1.73 ms in four rounds, 1.81 in one, whose keys do not stay in the L2.
// Work of less than two such rounds is one round: each cut tile costs a join.
constexpr int kRoundUnits = 100, kMaxRounds = 4;
constexpr int kTmaWarp = 8, kMmaWarp = 9, kWalkWarp = 10, kFixWarp = 11, kThreads = 384;
constexpr int kQueue = 4, kReaders = 11;              // steps of work handed on at a time, to 8 softmax warps, TMA, MMA and the fixing warp
// registers a thread: 384 x 168 at launch = 128 x kOtherRegs + 256 x kSoftRegs
constexpr int kSoftRegs = 216, kOtherRegs = 72;
// A weight is 2^(c s - m) by one fused operation, and the rounding of the reference m is a factor that all weights of a row share.  It is at most 2^0.5
// up to m = 2^24; beyond, it would carry p out of fp16's range and then out of a float's.  So m is kept to that by halving the row's c, as often as the
// maximum itself asks for: scores are then held to a step of 1 where they have a step of 1 or more in fp32 anyway.  (The reference is then moved without
// a lag, which would be one of halved units: parts compare their references in whole ones.)
constexpr float kLargeScore = 16777216.f;
constexpr long long kWaitCycles = 2000000000ll;       // about a second
constexpr long long kBeatCycles = 1 << 24;            // and as much for each stretch of 4096 keys that mend() has gone through: several times what it takes

__device__ int g_prompt_status;

struct PromptParams {
    void* out;                                        // [Tq, H, D]
    const void* q; const void* k; const void* v;      // only for what mend() does; the products read them through tensor maps
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;      // strides in elements
    const int32_t* cu_q; const int32_t* cu_k;
    int Tq, Tk, H, group, B;                          // group: query heads of a key head
    float scale_log2;                                 // |scale| * log2(e), above 0
    int negate;                                       // the scale is negative: the products with q are negated
    int causal;
    int most_rounds;                                  // that the scratch is made for
    // Where the line of work is cut inside a (head, tile), the pieces leave (O, m, l) in `partial`, two slots for a part of the line, and the last to
    // finish joins them.  counters: 8 for a part (that of the first piece; one for each softmax warp), zero between calls.
    float* partial;
    int* counters;
};

template <int D>
struct PromptCfg {
    static constexpr uint32_t kBox = 64 * 2 * kTileK;                       // 64 values x 128 rows
    static constexpr uint32_t kTileBytes = kBox * (D / 64);
    static constexpr int kSlots = D == 128 ? 4 : 8;                         // ring of K and V tiles
    static constexpr uint32_t kQOff = 0, kRingOff = 2 * kTileBytes, kBarOff = kRingOff + kSlots * kTileBytes;
    static constexpr uint32_t kQueueOff = kBarOff + 384;                    // kQueue steps of work
    static constexpr uint32_t kStageOff = kQueueOff + kQueue * 64;          // 32 rows x 32 finished values for each softmax warp
    static constexpr uint32_t kSmem = kStageOff + 8 * 2048 + 1024;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (abort_flag[0] != 0 || clock64() - t0 > kWaitCycles + abort_flag[1] * kBeatCycles) return false;
    return true;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// The same value from every lane, known to the compiler as such: it then lives in a uniform register, which is where
// tcgen05.mma takes its operands from (moving them there one by one was measured to cost twice the products' own time).
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(hi) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(hi) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
#define CB_R32(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7]), \
    "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]), "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), \
    "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]), "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), \
    "=r"(v[o + 24]), "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]), "=r"(v[o + 31])
#define CB_W32(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7]), \
    "r"(v[o + 8]), "r"(v[o + 9]), "r"(v[o + 10]), "r"(v[o + 11]), "r"(v[o + 12]), "r"(v[o + 13]), "r"(v[o + 14]), "r"(v[o + 15]), \
    "r"(v[o + 16]), "r"(v[o + 17]), "r"(v[o + 18]), "r"(v[o + 19]), "r"(v[o + 20]), "r"(v[o + 21]), "r"(v[o + 22]), "r"(v[o + 23]), \
    "r"(v[o + 24]), "r"(v[o + 25]), "r"(v[o + 26]), "r"(v[o + 27]), "r"(v[o + 28]), "r"(v[o + 29]), "r"(v[o + 30]), "r"(v[o + 31])
// 32 columns of this warp's lane quadrant, from column `addr` on, into v[O ..] / from v[O ..]
template <int O, int N> __device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[N]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : CB_R32(v, O) : "r"(addr));
}
template <int N> __device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[N]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                   "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
template <int O, int N> __device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[N]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(addr), CB_W32(v, O) : "memory");
}
#define CB_X32(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7]), \
    "+r"(v[o + 8]), "+r"(v[o + 9]), "+r"(v[o + 10]), "+r"(v[o + 11]), "+r"(v[o + 12]), "+r"(v[o + 13]), "+r"(v[o + 14]), "+r"(v[o + 15]), \
    "+r"(v[o + 16]), "+r"(v[o + 17]), "+r"(v[o + 18]), "+r"(v[o + 19]), "+r"(v[o + 20]), "+r"(v[o + 21]), "+r"(v[o + 22]), "+r"(v[o + 23]), \
    "+r"(v[o + 24]), "+r"(v[o + 25]), "+r"(v[o + 26]), "+r"(v[o + 27]), "+r"(v[o + 28]), "+r"(v[o + 29]), "+r"(v[o + 30]), "+r"(v[o + 31])
// All loads of this thread have arrived; v[O .. O + 31] are named so that nothing that uses them moves ahead of the wait.
template <int O, int N> __device__ __forceinline__ void tmem_ld_wait32(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : CB_X32(v, O) :: "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The work: all (head, tile of 256 query rows) pairs, sequence after sequence, tiles innermost, form one line of key tiles (and kOpen more ahead of each
// pair's) that is cut into equal parts: `rounds` for each CTA, CTA i taking parts i, i + CTAs, ...  In a round all CTAs are in one stretch of the
// line, a few heads wide, whose keys and values the L2 holds.  One warp walks through the CTA's parts, a few steps ahead, and hands the steps to the
// others through a queue in shared memory.
struct Work {                                         // head < 0: the end
    int head, row0, lq, lk, q_first, k_first;         // row0: the tile's first query row in its sequence; k_first, lk: from this part's first key on
    int n[2];                                         // key tiles of the sub-tiles, in this part
    int parts, slot, first, odd0;                     // pieces of this tile and head; this one's slot of scratch; piece i's is (first + i) * 2 (+ odd0 for i = 0)
};
struct Walk {
    int64_t u, u0, u1, base, share, extra;            // the present part [u0, u1) of the line; base: the present sequence's first unit
    int part, rounds, b, lq, lk, q_first, k_first;
};
__device__ __forceinline__ int row_range(const int32_t* cu, int b, int rows, int& first) {
    const int s = min(max(cu[b], 0), rows), e = min(max(cu[b + 1], s), rows);
    first = s;
    return e - s;
}
// Key tiles that the `rows` query rows from r0 on see together.
__device__ __forceinline__ int key_tiles(const PromptParams& P, int r0, int rows, int lq, int lk) {
    int64_t n = lk;
    if (P.causal) n = min(n, (int64_t)r0 + rows + (lk - lq));
    return rows <= 0 || n <= 0 ? 0 : (int)((n + kTileK - 1) / kTileK);
}
// a / b, both not negative, mostly by the much shorter 32-bit division.
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
    return a / b;
}
// Units of the first t tiles of a head of a sequence.  Under the causal bound tile i (of 256 rows) sees 2 (i + 1) + o key tiles, o = ceil((lk - lq) / 128),
// or none; only the last tile may have fewer rows.
__device__ __forceinline__ int64_t units_before(const PromptParams& P, int t, int lq, int lk) {
    const int tiles = (int)(((int64_t)lq + kTileQ - 1) / kTileQ), full = min(t, tiles - 1);
    int64_t n = 0;
    if (!P.causal) n = (int64_t)full * key_tiles(P, 0, 1, lq, lk);
    else {
        const int64_t off = (int64_t)lk - lq, o = off >= 0 ? (off + kTileK - 1) / kTileK : -(-off / kTileK);
        const int64_t from = o < 0 ? min(-o / 2, (int64_t)full) : 0;      // tiles before it see nothing
        n = ((int64_t)full * (full + 1) - from * (from + 1)) + (full - from) * o;
    }
    if (t >= tiles && tiles > 0) n += key_tiles(P, (tiles - 1) * kTileQ, lq - (tiles - 1) * kTileQ, lq, lk);
    return n + (int64_t)kOpen * max(t, 0);
}
__device__ __forceinline__ int64_t units_of(const PromptParams& P, int lq, int lk) {
    return lq <= 0 ? 0 : units_before(P, (int)(((int64_t)lq + kTileQ - 1) / kTileQ), lq, lk) * P.H;
}

// All lanes of a warp call these together.  false: there is nothing (more) to do.
__device__ __forceinline__ bool walk_part(const PromptParams& P, int lane, Walk& walk, int part) {
    const int64_t c = part, u0 = walk.share * c + min(c, walk.extra), u1 = walk.share * (c + 1) + min(c + 1, walk.extra);
    walk.part = part;
    int64_t base = 0;
    for (int b0 = 0; b0 < P.B; b0 += 32) {
        int first_q = 0, first_k = 0;
        const int b = b0 + lane;
        const int lq = b < P.B ? row_range(P.cu_q, b, P.Tq, first_q) : 0, lk = b < P.B ? row_range(P.cu_k, b, P.Tk, first_k) : 0;
        const int64_t mine = units_of(P, lq, lk);
        int64_t cum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, cum, o);
            if (lane >= o) cum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + cum > u0);
        if (past != 0u) {
            const int l = __ffs(past) - 1;
            walk.u = walk.u0 = u0; walk.u1 = u1;
            walk.base = base + __shfl_sync(0xffffffffu, cum - mine, l);
            walk.b = b0 + l;
            walk.lq = __shfl_sync(0xffffffffu, lq, l); walk.lk = __shfl_sync(0xffffffffu, lk, l);
            walk.q_first = __shfl_sync(0xffffffffu, first_q, l); walk.k_first = __shfl_sync(0xffffffffu, first_k, l);
            return true;
        }
        base += __shfl_sync(0xffffffffu, cum, 31);
    }
    return false;
}
__device__ __forceinline__ bool walk_begin(const PromptParams& P, int lane, Walk& walk) {
    int64_t U = 0;
    for (int b = lane; b < P.B; b += 32) {
        int first;
        U += units_of(P, row_range(P.cu_q, b, P.Tq, first), row_range(P.cu_k, b, P.Tk, first));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) U += __shfl_xor_sync(0xffffffffu, U, o);
    const int rounds = (int)min(max(div64(U, (int64_t)gridDim.x * kRoundUnits), (int64_t)1), (int64_t)P.most_rounds);
    const int64_t nc = min((int64_t)gridDim.x * rounds, U);
    if ((int64_t)blockIdx.x >= nc) return false;
    const int64_t share = nc == 0 ? 0 : div64(U, nc), extra = U - share * nc;
    walk.share = share; walk.extra = extra; walk.rounds = rounds;
    return walk_part(P, lane, walk, blockIdx.x);
}
__device__ __forceinline__ bool walk_next(const PromptParams& P, int lane, Walk& walk, Work& w) {
    for (;;) {
        if (walk.u >= walk.u1) {                      // the next round's part
            const int64_t part = (int64_t)walk.part + gridDim.x;
            if (part >= (int64_t)gridDim.x * walk.rounds || !walk_part(P, lane, walk, (int)part)) return false;
        }
        const int64_t u = walk.u;
        for (int64_t n = units_of(P, walk.lq, walk.lk); u >= walk.base + n; n = units_of(P, walk.lq, walk.lk)) {
            walk.base += n;
            if (++walk.b >= P.B) return false;        // only if the bounds changed while the kernel ran
            walk.lq = row_range(P.cu_q, walk.b, P.Tq, walk.q_first);
            walk.lk = row_range(P.cu_k, walk.b, P.Tk, walk.k_first);
        }
        const int lq = walk.lq, lk = walk.lk;
        int lo = 0, hi = (int)(((int64_t)lq + kTileQ - 1) / kTileQ);
        const int64_t each = units_before(P, hi, lq, lk);                 // of a head
        w.head = (int)div64(u - walk.base, each);
        const int64_t local = u - walk.base - w.head * each;
        while (hi - lo > 1) {                         // the tile: units_before(lo) <= local < units_before(hi)
            const int mid = (lo + hi) >> 1;
            if (units_before(P, mid, lq, lk) <= local) lo = mid; else hi = mid;
        }
        w.row0 = lo * kTileQ;
#pragma unroll
        for (int x = 0; x < 2; ++x) w.n[x] = key_tiles(P, w.row0 + x * kSub, min(lq - w.row0 - x * kSub, kSub), lq, lk);
        const int n = max(w.n[0], w.n[1]), per = n + kOpen;
        const int at = (int)(local - units_before(P, lo, lq, lk)), j0 = max(at - kOpen, 0);
        const int64_t seg0 = u - at;
        const int j1 = (int)min((int64_t)n, walk.u1 - seg0 - kOpen);
        walk.u = seg0 + per;
        if (n == 0 ? at > 0 : j1 <= j0) continue;     // rows without keys belong to the part with their first unit; of others this is the opening only
        w.lq = lq; w.q_first = walk.q_first;
        w.lk = lk - j0 * kTileK; w.k_first = walk.k_first + j0 * kTileK;
        w.parts = 1; w.slot = w.first = w.odd0 = 0;
        if (n > 0 && (j0 > 0 || j1 < n)) {
            const int64_t share = walk.share, extra = walk.extra;
            auto part_of = [&](int64_t unit) { return unit < extra * (share + 1) ? div64(unit, share + 1) : extra + div64(unit - extra * (share + 1), share); };
            const int64_t p0 = part_of(seg0 + kOpen);
            w.first = (int)p0;
            w.parts = (int)(part_of(seg0 + per - 1) - p0) + 1;
            w.slot = walk.part * 2 + (u == walk.u0 ? 0 : 1);
            w.odd0 = share * p0 + min(p0, extra) < seg0 ? 1 : 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) w.n[x] = min(max(w.n[x] - j0, 0), j1 - j0);
        }
        return true;
    }
}

__device__ __forceinline__ int arrive(int* counter) {
    int before;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16-bit values d .. d + 7 of a row times those of another, added up in four sums.
template <typename T> __device__ __forceinline__ void dot8(const uint4& a, const uint4& b, float (&s)[4]) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = unpack2<T>(x[i]), v = unpack2<T>(y[i]);
        s[i] = fmaf(u.x, v.x, fmaf(u.y, v.y, s[i]));
    }
}

// Is there a value that is not finite among keys [from, end) of the step?  The warp looks together, D / 32 columns to a lane.
template <typename T, int D>
__device__ __forceinline__ bool any_not_finite(const PromptParams& P, int lane, int head, int64_t k_first, int from, int end) {
    const T* val = reinterpret_cast<const T*>(P.v) + k_first * P.v_tok + (head / P.group) * P.v_head + lane * (D / 32);
    bool found = false;
#pragma unroll 8
    for (int key = from; key < end; ++key) {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(val + key * P.v_tok);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            const float2 f = unpack2<T>(at[i]);
            found = found || !(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY);
        }
    }
    return __any_sync(0xffffffffu, found);
}

// One row, as this warp has just stored it: finished at `out` (O times inv), or O itself at `part` (column c at part[c * kSub]).  If a key of the row's key
// tiles that the row does not see holds a value that is not finite in a column that came out as NaN, the column's sum over the keys that the row
// does see is formed again: keys [0, limit) of the step.  The warp does this together, a key to a lane for the weights, D / 32 columns to a lane for the
// sums; about 100 ns a key.  `beat` counts its stretches, for those who wait for this warp.  (As a call it is 0.2 us slower where it is not called.)
template <typename T, int D>
__device__ __forceinline__ void mend(const PromptParams& P, int lane, int head, int64_t q_row, int64_t k_first, int limit, int end, float factor, float m_ref,
                                  float inv, T* out, float* part, int* beat) {
    constexpr int kV = D / 32;
    const int64_t kv_head = head / P.group;
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(P.q) + q_row * P.q_tok + head * P.q_head);
    const T* k = reinterpret_cast<const T*>(P.k) + k_first * P.k_tok + kv_head * P.k_head;
    const T* val = reinterpret_cast<const T*>(P.v) + k_first * P.v_tok + kv_head * P.v_head + lane * kV;
    auto values = [&](int key, float (&x)[kV]) {                  // this lane's columns of a key's values
        const uint32_t* at = reinterpret_cast<const uint32_t*>(val + key * P.v_tok);
#pragma unroll
        for (int i = 0; i < kV / 2; ++i) { const float2 f = unpack2<T>(at[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    };
    uint32_t spoilt = 0u;
#pragma unroll 4
    for (int key = limit; key < end; ++key) {
        float x[kV];
        values(key, x);
#pragma unroll
        for (int i = 0; i < kV; ++i)
            if (!(fabsf(x[i]) < INFINITY)) spoilt |= 1u << i;
    }
    float v[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        v[i] = out != nullptr ? to_f32(*reinterpret_cast<const volatile T*>(out + lane * kV + i)) : __ldcg(part + (lane * kV + i) * kSub);
        if (v[i] == v[i]) spoilt &= ~(1u << i);
        v[i] = 0.f;
    }
    if (!__any_sync(0xffffffffu, spoilt != 0u)) return;
    const float neg = m_ref == -INFINITY ? 0.f : -m_ref, mul = P.negate ? -factor : factor;
    for (int key0 = 0; key0 < limit; key0 += 32) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (key0 + lane < limit) {
            const uint4* row = reinterpret_cast<const uint4*>(k + (key0 + lane) * P.k_tok);
#pragma unroll
            for (int d = 0; d < D / 8; ++d) dot8<T>(q[d], row[d], s);
        }
        const float p = ex2(fmaf((s[0] + s[1]) + (s[2] + s[3]), mul, neg));
        const int n = min(limit - key0, 32);
        if (n == 32) {
#pragma unroll 16
            for (int i = 0; i < 32; ++i) {
                float x[kV];
                values(key0 + i, x);
                const float pi = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
                for (int c = 0; c < kV; ++c) v[c] = fmaf(pi, x[c], v[c]);
            }
        } else
            for (int i = 0; i < n; ++i) {
                float x[kV];
                values(key0 + i, x);
                const float pi = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
                for (int c = 0; c < kV; ++c) v[c] = fmaf(pi, x[c], v[c]);
            }
        if ((key0 & 4095) == 0 && lane == 0) atomicAdd(beat, 1);
        bool open = false;                                        // NaN stays: the row may see one itself
#pragma unroll
        for (int c = 0; c < kV; ++c) open = open || (((spoilt >> c) & 1u) && v[c] == v[c]);
        if (!__any_sync(0xffffffffu, open)) break;
    }
#pragma unroll
    for (int i = 0; i < kV; ++i)
        if ((spoilt >> i) & 1u) {
            if (out != nullptr) out[lane * kV + i] = from_f32<T>(v[i] * inv);
            else __stcg(part + (lane * kV + i) * kSub, v[i]);
        }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PromptParams P) {
    using C = PromptCfg<D>;
    constexpr int kSlots = C::kSlots;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars = base + C::kBarOff;
    auto q_full = [&](int x) { return bars + 8u * x; };
    const uint32_t q_empty = bars + 16u;
    auto s_full = [&](int x) { return bars + 24u + 8u * x; };
    auto p_ready = [&](int x, int half) { return bars + 40u + 16u * x + 8u * half; };
    auto pv_done = [&](int x) { return bars + 72u + 8u * x; };
    auto o_free = [&](int x) { return bars + 88u + 8u * x; };
    const uint32_t v_landed = bars + 104u, v_fixed = bars + 112u;
    auto kv_full = [&](int s) { return bars + 120u + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 120u + 8u * (kSlots + s); };
    auto w_full = [&](uint32_t i) { return bars + 256u + 8u * (i % kQueue); };
    auto w_empty = [&](uint32_t i) { return bars + 256u + 8u * (kQueue + i % kQueue); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::kBarOff + 352);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kBarOff + 356);        // [1]: stretches of mend()
    volatile uint32_t* copied = reinterpret_cast<volatile uint32_t*>(smem + C::kBarOff + 364);       // K and V tiles, and tiles of Q, that copies were issued for
    const uint32_t drained = bars + 376u;
    static_assert(120 + 16 * kSlots <= 256 && 256 + 16 * kQueue <= 352 && C::kQueueOff >= C::kBarOff + 384, "barriers");
    Work* queue = reinterpret_cast<Work*>(smem + C::kQueueOff);
    static_assert(sizeof(Work) <= 64, "a step of work");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; ++x) {
            mbar_init(q_full(x), 1); mbar_init(s_full(x), 1); mbar_init(p_ready(x, 0), 4); mbar_init(p_ready(x, 1), 4); mbar_init(pv_done(x), 1); mbar_init(o_free(x), 4);
        }
        for (int i = 0; i < kQueue; ++i) { mbar_init(w_full(i), 1); mbar_init(w_empty(i), kReaders); }
        mbar_init(q_empty, 1); mbar_init(drained, 1); mbar_init(v_landed, 1); mbar_init(v_fixed, 1);
        for (int s = 0; s < kSlots; ++s) { mbar_init(kv_full(s), 1); mbar_init(kv_empty(s), 1); }
        abort_flag[0] = abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((const void*)tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    int gave_up = 0;

    // The steps of work, as a reader sees them: next() waits for one, done() hands it back.
    uint32_t step = 0;
    const Work* wp = queue;
    auto next = [&]() {
        if (gave_up) return false;
        if (!__all_sync(0xffffffffu, mbar_wait(w_full(step), (step / kQueue) & 1, abort_flag))) { gave_up = 6; return false; }
        wp = queue + step % kQueue;
        return wp->head >= 0;
    };
    auto done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(w_empty(step));
        ++step;
    };
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kWalkWarp) {
        // ================= the walk =================
        Walk walk;
        Work w;
        bool more = walk_begin(P, lane, walk);
        for (; !gave_up; ++step) {
            more = more && walk_next(P, lane, walk, w);
            if (!more) w.head = -1;
            if (step >= kQueue && !__all_sync(0xffffffffu, mbar_wait(w_empty(step), (step / kQueue - 1) & 1, abort_flag))) { gave_up = 6; break; }
            if (lane == 0) {
                queue[step % kQueue] = w;
                mbar_arrive(w_full(step));
            }
            __syncwarp();
            if (!more) break;
        }
    } else if (warp == kTmaWarp) {
        // ================= TMA: Q once a tile, K and V tiles through the ring =================
        uint32_t it = 0, tiles = 0;
        for (; next(); done()) {
            const Work w = *wp;
            const int n = max(w.n[0], w.n[1]);
            if (n == 0) continue;
            if (tiles > 0 && !__all_sync(0xffffffffu, mbar_wait(q_empty, (tiles - 1) & 1, abort_flag))) { gave_up = 1; break; }
            ++tiles;
            const int kv_head = w.head / P.group;
            if (lane == 0)
                for (int x = 0; x < 2; ++x) {
                    mbar_expect_tx(q_full(x), C::kTileBytes);
                    for (int h = 0; h < D / 64; ++h)
                        tma_load_3d(base + C::kQOff + x * C::kTileBytes + h * C::kBox, &qmap, h * 64, w.head, w.q_first + w.row0 + x * kSub, q_full(x));
                }
            for (int j = 0; j < 2 * n; ++j, ++it) {               // K tile, V tile, K tile, ...
                const int s = it % kSlots;
                if (it >= kSlots && !__all_sync(0xffffffffu, mbar_wait(kv_empty(s), (it / kSlots - 1) & 1, abort_flag))) { gave_up = 1; break; }
                if (lane == 0) {
                    mbar_expect_tx(kv_full(s), C::kTileBytes);
                    for (int h = 0; h < D / 64; ++h)
                        tma_load_3d(base + C::kRingOff + s * C::kTileBytes + h * C::kBox, (j & 1) ? &vmap : &kmap, h * 64, kv_head,
                                    w.k_first + (j >> 1) * kTileK, kv_full(s));
                }
            }
        }
        if (lane == 0) { copied[0] = it; copied[1] = tiles; }
    } else if (warp == kMmaWarp) {
        // ================= MMA issuer: the warp goes through the list together, one elected thread issues =================
        constexpr uint32_t fmt = BF ? ((1u << 7) | (1u << 10)) : 0u;
        const uint32_t idesc_s = (1u << 4) | fmt | ((uint32_t)P.negate << 13) | ((uint32_t)(kTileK >> 3) << 17) | ((uint32_t)(kSub >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | fmt | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kSub >> 4) << 24);
        constexpr uint64_t dk = (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);                        // K-major, 128-byte swizzle, 8-row atoms 1024 bytes apart
        constexpr uint64_t dv = ((uint64_t)(C::kBox >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);    // N-major: 64-value boxes kBox apart, 8-key groups 1024 bytes apart
        const uint32_t tm = uniform(tmem), ring = uniform((base + C::kRingOff) >> 4), q_at = uniform((base + C::kQOff) >> 4);
        uint32_t it = 0, tiles = 0, fixes = 0, pcount[2] = {0, 0}, ocount[2] = {0, 0};
        // the ring place of K tile j of the present query tile is it + 2 j, of V tile j it + 2 j + 1
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag))) gave_up = 2;
            return gave_up == 0;
        };
        auto scores = [&](int x, uint32_t place, bool release) {
            const uint32_t slot = place % kSlots;
            const uint32_t ad = (uint32_t)dk | (q_at + x * (C::kTileBytes >> 4)), bd = (uint32_t)dk | (ring + slot * (C::kTileBytes >> 4));
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    constexpr uint32_t kBox16 = C::kBox >> 4;
                    const uint32_t off = (k / 4) * kBox16 + (k % 4) * 2;
                    mma_ss(tm + x * 128, ad + off, bd + off, (uint32_t)(dk >> 32), idesc_s, k > 0 ? 1u : 0u);
                }
                commit(s_full(x));
                if (release) commit(kv_empty(slot));
            }
            __syncwarp();
        };
        auto values = [&](int x, uint32_t place, bool first, bool release) {
            const uint32_t slot = place % kSlots;
            const uint32_t bd = (uint32_t)dv | (ring + slot * (C::kTileBytes >> 4));
#pragma unroll
            for (int half = 0; half < 2; ++half) {                // the first 64 keys' product while the others' weights are made
                if (!wait(p_ready(x, half), pcount[x] & 1)) return;
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k4 = 0; k4 < kTileK / 32; ++k4) {
                        const int k = half * (kTileK / 32) + k4;
                        mma_ts(tm + 256 + x * 128, tm + x * 128 + k * 8, bd + k * 128, (uint32_t)(dv >> 32), idesc_o, first && k == 0 ? 0u : 1u);
                    }
                    if (half == 1) {
                        commit(pv_done(x));
                        if (release) commit(kv_empty(slot));
                    }
                }
                __syncwarp();
            }
            ++pcount[x];
        };
        for (; next(); done()) {
            const Work& w = *wp;
            const int n0 = (int)uniform(w.n[0]), n1 = (int)uniform(w.n[1]), lk = (int)uniform(w.lk), n = max(n0, n1);
            if (n == 0) continue;
            // both halves of Q are always loaded
            if (!wait(q_full(0), tiles & 1) || !wait(q_full(1), tiles & 1) || !wait(kv_full(it % kSlots), (it / kSlots) & 1)) break;
            ++tiles;
            fence_after();
            if (n0 > 0) scores(0, it, n1 == 0);
            if (n1 > 0) scores(1, it, true);
            if (n == 1 && elect_one()) commit(q_empty);           // the last scores: the next tile's Q may come
            for (int j = 0; j < n && !gave_up; ++j) {
                const uint32_t v = it + 2 * j + 1, k = v + 1;
                if (!wait(kv_full(v % kSlots), (v / kSlots) & 1)) break;
                if (lk - j * kTileK < kTileK) {
                    if (lane == 0) mbar_arrive(v_landed);         // only now: the fixing warp does not follow the ring itself
                    if (!wait(v_fixed, fixes++ & 1)) break;
                }
                if (j + 1 < n && !wait(kv_full(k % kSlots), (k / kSlots) & 1)) break;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int nx = x == 0 ? n0 : n1;
                    if (j < nx) {
                        if (j == 0) {                             // the previous tile's O must have been read
                            if (ocount[x] > 0 && !wait(o_free(x), (ocount[x] - 1) & 1)) break;
                            ++ocount[x];
                        }
                        values(x, v, j == 0, x == 1 || j >= n1);
                    }
                    if (gave_up) break;
                    if (j + 1 < nx) scores(x, k, x == 1 || j + 1 >= n1);
                }
                if (j + 2 == n && !gave_up && elect_one()) commit(q_empty);
                __syncwarp();
            }
            it += 2 * n;
        }
    } else if (warp == kFixWarp) {
        // ================= the last V tile of a sequence: zeros behind its last key, before any product reads it =================
        uint32_t it = 0, fixes = 0;
        for (; next(); done()) {
            const Work& w = *wp;
            const int n = max(w.n[0], w.n[1]), valid = w.lk - (n - 1) * kTileK;
            if (n == 0) continue;
            it += 2 * n;
            if (valid >= kTileK) continue;
            const uint32_t place = it - 1;
            if (!__all_sync(0xffffffffu, mbar_wait(v_landed, fixes++ & 1, abort_flag))) { gave_up = 5; break; }
            unsigned char* v = smem + C::kRingOff + (place % kSlots) * C::kTileBytes;
            for (int i = lane; i < (kTileK - valid) * 8; i += 32)
                for (int h = 0; h < D / 64; ++h) *reinterpret_cast<uint4*>(v + h * C::kBox + valid * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(v_fixed);
        }
    }
    } else {
        // ================= softmax and epilogue: a thread owns a row =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int x = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16), s_addr = lane_base + x * 128, o_addr = lane_base + 256 + x * 128;
        uint32_t count = 0;                                       // score tiles of this sub-tile so far
        for (; next(); done()) {
            const Work& w = *wp;
            const int n = w.n[x], r = w.row0 + x * kSub + row;    // query row in its sequence
            const bool live = r < w.lq;
            T* dst = reinterpret_cast<T*>(P.out) + ((int64_t)(w.q_first + r) * P.H + w.head) * D;
            if (n == 0 && w.parts == 1) {                         // rows that see no key
                if (live)
                    for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0u, 0u, 0u, 0u);
                continue;
            }
            const int limit = P.causal ? (int)min((int64_t)w.lk, max((int64_t)0, (int64_t)r + 1 + w.lk - w.lq)) : w.lk;      // keys this row sees
            float m_ref = -INFINITY, l = 0.f, factor = P.scale_log2, lag = 8.f;
            for (int j = 0; j < n; ++j, ++count) {
                if (!__all_sync(0xffffffffu, mbar_wait(s_full(x), count & 1, abort_flag))) { gave_up = 3; break; }
                fence_after();
                uint32_t s[128];
                tmem_ld32<0>(s_addr, s); tmem_ld32<32>(s_addr + 32, s);
                tmem_ld_wait32<0>(s); tmem_ld_wait32<32>(s);
                tmem_ld32<64>(s_addr + 64, s); tmem_ld32<96>(s_addr + 96, s);
                const int seen = limit - j * kTileK;
                const bool masked = __any_sync(0xffffffffu, seen < kTileK);
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (masked)
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (i >= seen) s[i] = 0xff800000u;
#pragma unroll
                for (int i = 0; i < 64; i += 8)
#pragma unroll
                    for (int c = 0; c < 4; ++c) m4[c] = fmaxf(m4[c], fmaxf(__uint_as_float(s[i + c]), __uint_as_float(s[i + 4 + c])));
                tmem_ld_wait32<64>(s); tmem_ld_wait32<96>(s);
                if (masked)
#pragma unroll
                    for (int i = 64; i < 128; ++i)
                        if (i >= seen) s[i] = 0xff800000u;
#pragma unroll
                for (int i = 64; i < 128; i += 8)
#pragma unroll
                    for (int c = 0; c < 4; ++c) m4[c] = fmaxf(m4[c], fmaxf(__uint_as_float(s[i + c]), __uint_as_float(s[i + 4 + c])));
                const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                float m = top * factor;
                const bool move = m > m_ref + lag;
                if (__any_sync(0xffffffffu, move)) {
                    if (move && (lag == 0.f || fabsf(m) > kLargeScore) && fabsf(top) < INFINITY) {
                        float mul = P.scale_log2;
                        for (m = top * mul; fabsf(m) > kLargeScore; m = top * mul) { mul *= 0.5f; lag = 0.f; }
                        m_ref *= mul / factor;
                        factor = mul;
                    }
                    const float a = move ? ex2(m_ref - m) : 1.f;
                    if (move) m_ref = m;
                    l *= a;
                    if (j > 0) {
                        if (!__all_sync(0xffffffffu, mbar_wait(pv_done(x), (count - 1) & 1, abort_flag))) { gave_up = 3; break; }
                        fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t v[32];
                            tmem_ld32<0>(o_addr + c, v);
                            tmem_ld_wait32<0>(v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
                            tmem_st32<0>(o_addr + c, v);
                        }
                        tmem_st_wait();
                    }
                }
                // ---- weights, 32 keys at a time
                const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
                const f32x2 neg2 = pair(neg, neg), mul = pair(factor, factor);
                f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t out[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float p0, p1;
                        unpair(fma2(pair(s[32 * c + 2 * i], s[32 * c + 2 * i + 1]), mul, neg2), p0, p1);
                        p0 = ex2(p0); p1 = ex2(p1);
                        sum[i & 1] = add2(sum[i & 1], pair(p0, p1));
                        out[i] = pack2<T>(p0, p1);
                    }
                    tmem_st16(s_addr + 16 * c, out);
                    if (c & 1) {
                        tmem_st_wait();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready(x, c >> 1));
                    }
                }
                float l0, l1;
                unpair(add2(sum[0], sum[1]), l0, l1);
                l += l0 + l1;
            }
            if (gave_up) break;
            if (n > 0) {
                if (!__all_sync(0xffffffffu, mbar_wait(pv_done(x), (count - 1) & 1, abort_flag))) { gave_up = 4; break; }
                fence_after();
            }
            // Of this part's keys this row sees none: its O is 0, whatever the values that met its weights of 0 are.  A row that sees keys has l = 0
            // only if all their scores are -inf, and l NaN if one is NaN or +inf: O / l is NaN then, as the definition has it.
            const bool blind = limit <= 0;
            // a cut tile: O[d][row], m[row], l[row] of this part and sub-tile; l is -1, and O anything, where the row is blind
            constexpr int kPart = kSub * (D + 2);
            auto slot_at = [&](int slot) { return P.partial + ((int64_t)slot * 2 + x) * kPart + row; };
            auto part_at = [&](int i) { return slot_at((w.first + i) * 2 + (i == 0 ? w.odd0 : 0)); };
            const float inv = 1.f / l;
            // 32 finished values of every row of the warp: turned over in shared memory, so that a store covers 64 contiguous bytes of each of 8 rows (a
            // lane's own row, 16 bytes at a time, takes a line for each lane: the stores of a tile were then 2 us).  Pieces of 16 bytes stand
            // where eight lanes that write or read together meet different banks.
            auto store32 = [&](int c, const uint32_t (&v)[32]) {
                unsigned char* stage = smem + C::kStageOff + warp * 2048;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        y[k] = blind ? 0u : pack2<T>(__uint_as_float(v[8 * i + 2 * k]) * inv, __uint_as_float(v[8 * i + 2 * k + 1]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int of = i * 8 + (lane >> 2), piece = lane & 3, at = w.row0 + x * kSub + quad * 32 + of;      // another lane's row
                    const uint4 y = *reinterpret_cast<const uint4*>(stage + of * 64 + ((piece ^ ((of >> 1) & 3)) * 16));
                    if (at < w.lq)
                        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(P.out) + ((int64_t)(w.q_first + at) * P.H + w.head) * D + c + piece * 8) = y;
                }
            };
            auto put32 = [&](int c, const uint32_t (&v)[32]) {
                if (w.parts == 1) store32(c, v);
                else {
                    float* at = slot_at(w.slot) + c * kSub;
#pragma unroll
                    for (int i = 0; i < 32; ++i) __stcg(at + i * kSub, __uint_as_float(v[i]));
                }
            };
            if (n > 0) {
                f32x2 sums[2] = {0ull, 0ull};                     // not finite if a value is not
                // not unrolled, as little here is: code that runs once a tile comes from afar each time, and was measured to cost more than its work
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t v[32];
                    tmem_ld32<0>(o_addr + c, v);
                    tmem_ld_wait32<0>(v);
                    if (c + 32 == D) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(o_free(x));
                    }
                    put32(c, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[i & 1] = add2(sums[i & 1], pair(v[2 * i], v[2 * i + 1]));
                }
                float s0, s1;
                unpair(add2(sums[0], sums[1]), s0, s1);
                __syncwarp();                                     // other lanes have stored this row
                unsigned left = __ballot_sync(0xffffffffu, !(fabsf(s0 + s1) < INFINITY) && live && !blind && l == l);
                // (that the rows see such values themselves is the commoner case)
                if (left != 0u && !any_not_finite<T, D>(P, lane, w.head, w.k_first, __shfl_sync(0xffffffffu, limit, __ffs(left) - 1), min(n * kTileK, w.lk))) left = 0u;
                for (; left != 0u; left &= left - 1u) {
                    const int of = __ffs(left) - 1, at = w.row0 + x * kSub + quad * 32 + of;      // the row of another lane
                    const float f = __shfl_sync(0xffffffffu, factor, of), m = __shfl_sync(0xffffffffu, m_ref, of), i = __shfl_sync(0xffffffffu, inv, of);
                    const int see = __shfl_sync(0xffffffffu, limit, of);
                    mend<T, D>(P, lane, w.head, w.q_first + at, w.k_first, see, min(n * kTileK, w.lk), f, m, i,
                               w.parts == 1 ? reinterpret_cast<T*>(P.out) + ((int64_t)(w.q_first + at) * P.H + w.head) * D : nullptr, slot_at(w.slot) - lane + of, const_cast<int*>(abort_flag) + 1);
                }
            }
            if (w.parts == 1) continue;
            __stcg(slot_at(w.slot) + D * kSub, lag == 0.f ? m_ref * (P.scale_log2 / factor) : m_ref);
            __stcg(slot_at(w.slot) + (D + 1) * kSub, blind ? -1.f : l);
            __syncwarp();
            int last = 0;
            if (lane == 0) {
                int* counter = P.counters + (w.first * 2 + x) * 4 + quad;
                // this warp's rows, ordered before by its barrier, are visible to who sees the count, and the others' to this warp if it is the last
                last = arrive(counter) == w.parts - 1;
                if (last) *counter = 0;
            }
            last = __shfl_sync(0xffffffffu, last, 0);
            __syncwarp();
            if (last == 0) continue;
            // this warp's rows are complete in all parts: joined in their order.  Parts that are blind count for nothing; one with a sum of NaN makes the
            // row NaN, as do scores of -inf in all that are not (top - top is NaN).
            float top = -INFINITY, sum = 0.f;
            for (int i = 0; i < w.parts; ++i) top = fmaxf(top, __ldcg(part_at(i) + D * kSub));
            for (int i = 0; i < w.parts; ++i) {
                const float m = __ldcg(part_at(i) + D * kSub), s = __ldcg(part_at(i) + (D + 1) * kSub);
                if (!(s < 0.f)) sum = fmaf(ex2(m - top), s, sum);
            }
            const float rsum = 1.f / sum;
#pragma unroll 1
            for (int c = 0; c < D; c += 64) {                     // 64 loads on their way at a time
                float v[64];
#pragma unroll
                for (int k = 0; k < 64; ++k) v[k] = 0.f;
#pragma unroll 1
                for (int i = 0; i < w.parts; ++i) {
                    const float* at = part_at(i);
                    const float m = __ldcg(at + D * kSub), s = __ldcg(at + (D + 1) * kSub);
                    float o[64];
#pragma unroll
                    for (int k = 0; k < 64; ++k) o[k] = __ldcg(at + (c + k) * kSub);
                    const float f = ex2(m - top) * rsum;
#pragma unroll
                    for (int k = 0; k < 64; ++k) v[k] = s < 0.f ? v[k] : fmaf(f, o[k], v[k]);
                }
                if (live)
#pragma unroll
                    for (int k = 0; k < 64; k += 8)
                        *reinterpret_cast<uint4*>(dst + c + k) = make_uint4(pack2<T>(v[k], v[k + 1]), pack2<T>(v[k + 2], v[k + 3]), pack2<T>(v[k + 4], v[k + 5]), pack2<T>(v[k + 6], v[k + 7]));
            }
        }
    }
    if (gave_up) {
        *abort_flag = 1;
        atomicExch(&g_prompt_status, gave_up);
    }
    fence_before();
    __syncthreads();
    if (*abort_flag != 0) {
        // Some role gave up, and others may have ended in good order before: copies and products that nobody waited for are still on their way into this
        // CTA's memory.  They are waited for, again with a limit, before it is given back.
        const long long t0 = clock64();
        auto drain = [&](uint32_t bar, uint32_t parity) { while (!mbar_try_wait(bar, parity) && clock64() - t0 < kWaitCycles) {} };
        if (warp == kTmaWarp) {
            const uint32_t it = copied[0], tiles = copied[1];
            for (uint32_t i = it > kSlots ? it - kSlots : 0; i < it; ++i) drain(kv_full(i % kSlots), (i / kSlots) & 1);
            for (int x = 0; x < 2 && tiles > 0; ++x) drain(q_full(x), (tiles - 1) & 1);
        }
        if (warp == kMmaWarp) {
            if (elect_one()) commit(drained);                     // by the thread that issued the products
            __syncwarp();
            drain(drained, 0);
            fence_before();
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

template <typename T, int D>
int launch_prompt_t(const CUtensorMap (&maps)[3], const PromptParams& P, int grid, cudaStream_t stream) {
    using C = PromptCfg<D>;
    static bool attr_done[64] = {};
    int dev = 0;
    CB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        CB_CUDA_TRY(cudaFuncSetAttribute(prompt_attention_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    prompt_attention_kernel<T, D><<<grid, kThreads, C::kSmem, stream>>>(maps[0], maps[1], maps[2], P);
    CB_CUDA_TRY(cudaGetLastError());
    return CB_OK;
}

}  // namespace

// Rounds that a call of these sizes may take: by the units that its sequences have at most (tiles, and key tiles of each), one CTA to an SM.
static int prompt_rounds(int64_t Tq, int64_t Tk, int64_t H, int64_t B, int sms) {
    const int64_t tiles = Tq / kTileQ + std::min(B, Tq), each = kOpen + (Tk + kTileK - 1) / kTileK;
    const int64_t enough = (int64_t)sms * kRoundUnits * kMaxRounds;          // H < 2^20, tiles and each < 2^31: the products are looked at one by one
    const int64_t per_head = tiles > enough / each ? enough : tiles * each;
    const int64_t units = per_head > enough / H ? enough : per_head * H;
    return (int)std::min<int64_t>(std::max<int64_t>(units / ((int64_t)sms * kRoundUnits), 1), kMaxRounds);
}
int64_t prompt_attention_most_parts() { return (int64_t)std::max(sm_count_current(), 0) * kMaxRounds; }
// Parts of the line, each of which may leave two pieces in scratch.  Up to kTileK keys a tile is one key tile, and never cut.
int64_t prompt_attention_parts(int64_t Tq, int64_t Tk, int64_t H, int64_t B) {
    const int sms = sm_count_current();
    return sms <= 0 || Tk <= kTileK ? 0 : (int64_t)sms * prompt_rounds(Tq, Tk, H, B, sms);
}
size_t prompt_attention_partial_bytes(int64_t parts, int head_dim) { return (size_t)parts * 2 * kTileQ * (head_dim + 2) * sizeof(float); }
size_t prompt_attention_counter_bytes(int64_t parts) { return (size_t)parts * 8 * sizeof(int); }

// Arguments are checked by the caller.  strides: {q token, q head, k token, k head, v token, v head} in elements.
int launch_prompt_attention(const void* q, const void* k, const void* v, const int64_t* strides, void* out, int64_t Tq, int64_t Tk,
                            int64_t H, int64_t Hkv, int head_dim, int dtype, const int32_t* cu_q, const int32_t* cu_k, int64_t B,
                            float scale, int causal, int* counters, float* partial, cudaStream_t stream) {
    const int sms = sm_count_current();
    if (sms <= 0) return CB_ERR_CUDA;
    EncodeTiledFn enc = encode_fn();
    if (enc == nullptr) { set_error("prompt_attention: cuTensorMapEncodeTiled is not available"); return CB_ERR_CUDA; }
    CUtensorMap maps[3];
    for (int i = 0; i < 3; ++i) {
        const bool none = i > 0 && Tk == 0;                       // no keys at all: a map that nothing is read through
        const void* p = i == 0 || none ? q : i == 1 ? k : v;
        const int64_t heads = i == 0 ? H : Hkv, rows = i == 0 ? Tq : none ? 1 : Tk;
        const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
        // the stride of a dimension of one entry is never used, but has to be a good one
        const cuuint64_t bytes[2] = {heads == 1 || none ? (cuuint64_t)head_dim * 2 : (cuuint64_t)strides[2 * i + 1] * 2,
                                     rows == 1 ? (cuuint64_t)head_dim * heads * 2 : (cuuint64_t)strides[2 * i] * 2};
        const cuuint32_t box[3] = {64, 1, 128}, step[3] = {1, 1, 1};
        const CUresult cr = enc(&maps[i], dtype == CB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                                const_cast<void*>(p), dims, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) { set_error("prompt_attention: cuTensorMapEncodeTiled(%c) failed (%d)", "qkv"[i], (int)cr); return CB_ERR_CUDA; }
    }
    PromptParams P{};
    P.out = out; P.cu_q = cu_q; P.cu_k = cu_k;
    P.q = q; P.k = k; P.v = v;
    P.q_tok = strides[0]; P.q_head = strides[1]; P.k_tok = strides[2]; P.k_head = strides[3]; P.v_tok = strides[4]; P.v_head = strides[5];
    P.Tq = (int)Tq; P.Tk = (int)Tk; P.H = (int)H; P.group = (int)(H / Hkv); P.B = (int)B;
    // a scale of 0 weighs all keys alike: the smallest float does (0 itself would make NaN of the -inf that stands for an unseen key)
    P.scale_log2 = scale == 0.f ? 1e-45f : std::min(fabsf(scale) * 1.4426950408889634f, FLT_MAX);
    P.negate = scale < 0.f ? 1 : 0;
    P.causal = causal ? 1 : 0;
    P.most_rounds = prompt_rounds(Tq, Tk, H, B, sms);
    P.counters = counters; P.partial = partial;
    const int grid = sms;
    const bool bf = dtype == CB_BF16;
    if (head_dim == 128) return bf ? launch_prompt_t<__nv_bfloat16, 128>(maps, P, grid, stream) : launch_prompt_t<__half, 128>(maps, P, grid, stream);
    return bf ? launch_prompt_t<__nv_bfloat16, 64>(maps, P, grid, stream) : launch_prompt_t<__half, 64>(maps, P, grid, stream);
}

int prompt_status_read_and_clear(int* out) {
    int v = 0, zero = 0;
    CB_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_prompt_status, sizeof(int)));
    CB_CUDA_TRY(cudaMemcpyToSymbol(g_prompt_status, &zero, sizeof(int)));
    *out = v;
    return CB_OK;
}

}  // namespace cb
