// Layout of the 4-bit key/value cache, shared by the kernels that write, read and attend to it.
//
// A group of GS values of one token and head is kept as lo (its smallest value), scale and GS codes of 4 bits:
// value = code * scale + lo.  lo and scale are of the cache's 16-bit type.
//
// The unit of storage is a BLOCK of 16 tokens of one head, contiguous:
//     K codes [16][D/2 bytes] | K meta [16][D/GS] (scale, lo) | V codes [16][D/2 bytes] | V meta [16][D/GS] (scale, lo)
// so that one bulk copy brings everything the attention of 16 tokens needs.  A page of a head is page_size / 16
// consecutive blocks, and pages are [n_pages][kv_heads][page].
//
// Inside a token's D/2 code bytes the values stand in the order in which the lanes of mma.sync fragments want them
// (a lane's codes are contiguous, one wide shared-memory load each):
//   * K is the A operand of S^T = K q^T.  Lane (r, t) of a fragment (r = lane / 4, t = lane % 4) takes the values
//     t * GS/4 .. t * GS/4 + GS/4 - 1 of every group, group after group.
//   * V is the A operand of O^T = V^T P^T.  Lane (r, t) takes the values r * GS/8 .. r * GS/8 + GS/8 - 1 of every
//     group.  At D = 128 the two 32-byte halves of a token whose number has bit 1 set are exchanged: the four tokens
//     that the lanes t = 0..3 read together then lie in different banks.
#pragma once
#include "cb_common.cuh"

namespace cb {

constexpr int kKvBlock = 16;      // tokens of a block

template <int D, int GS>
struct KvLayout {
    static constexpr int NG = D / GS;                          // groups of a row
    static constexpr int kRow = D / 2;                         // code bytes of a row
    static constexpr int kMeta = 4 * NG;                       // (scale, lo) bytes of a row
    static constexpr int kKMeta = kKvBlock * kRow;
    static constexpr int kVCodes = kKMeta + kKvBlock * kMeta;
    static constexpr int kVMeta = kVCodes + kKvBlock * kRow;
    static constexpr int kBytes = kVMeta + kKvBlock * kMeta;   // of a block

    // Number, inside its row, of the nibble that holds value d (a multiple of 8) of a key; the next 7 values follow.
    __host__ __device__ static constexpr int k_nibble(int d) {
        const int j = d / GS, w = d % GS;
        return (w / (GS / 4)) * (D / 4) + j * (GS / 4) + w % (GS / 4);
    }
    // The same for value d (a multiple of min(8, GS / 8)) of token `tok` (0..15) of V; the next min(8, GS / 8) follow.
    __host__ __device__ static constexpr int v_nibble(int d, int tok) {
        const int j = d / GS, w = d % GS;
        const int n = (w / (GS / 8)) * (D / 8) + j * (GS / 8) + w % (GS / 8);
        return D == 128 ? n ^ (((tok >> 1) & 1) << 6) : n;
    }
};

// What the kernels of the cache take of it.
struct Kv4View {
    unsigned char* pages;
    int64_t n_pages;
    int kv_heads, blocks_per_page;      // page_size / 16
    const int32_t* table;               // [n_seqs, table_stride] page numbers
    int64_t table_stride;
};

constexpr int kKv4BadPage = 3001;       // status word: a page number outside the cache was met and left out
constexpr int kKv4Wait = 3002;          // status word: a copy did not arrive in time

}  // namespace cb
