// Layout of the 4-bit key/value cache, shared by the kernels that write, read and attend to it.
//
// A group of GS values of one token and head is kept as lo (its smallest value), scale and GS codes of 4 bits:
// value = code * scale + lo.  lo and scale are of the cache's 16-bit type.
//
// The unit of storage is a BLOCK of 16 tokens of one head, contiguous:
//     K codes 16 x D/2 bytes | K meta [16][D/GS] (scale, lo) | V codes 16 x D/2 bytes | V meta [16][D/GS] (scale, lo)
// so that one bulk copy brings everything the attention of 16 tokens needs.  A page of a head is page_size / 16
// consecutive blocks, and pages are [n_pages][kv_heads][page].
//
// The codes stand in the order in which the lanes of mma.sync fragments want them (lane = 4 r + t):
//   * K is the 16-row operand of S^T = K q^T.  A token's D/2 bytes are contiguous; lane (r, t) takes the values
//     t * GS/4 .. t * GS/4 + GS/4 - 1 of every group, and they lie side by side: one wide shared-memory load.
//   * V is the 16-row operand of O^T = V^T P^T, whose registers hold the same value of two tokens: tokens t and 7 - t (t = 0..3),
//     and t + 8 and 15 - t.  Such a pair shares D bytes, in which lane r's D/8 bytes are the values
//     r * GS/8 .. r * GS/8 + GS/8 - 1 of every group, four at a time: 16 bits of the one token, 16 of the other.  The order of
//     the lanes' pieces depends on the pair such that lanes which read together meet different banks.
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
    // Byte, inside V's codes, of values d .. d + 3 (d a multiple of 4) of token `tok` (0..15): two bytes.
    __host__ __device__ static constexpr int v_byte(int d, int tok) {
        const int pair = ((tok & 4) ? 7 - (tok & 7) : (tok & 3)) + 4 * (tok >> 3);
        const int w = d % GS, lane = w / (GS / 8), unit = (d / GS * (GS / 8) + w % (GS / 8)) / 4;
        return pair * D + v_piece(lane, pair) + unit * 4 + ((tok & 4) ? 2 : 0);
    }
    // Where lane r's piece of a pair begins in the pair's D bytes.
    __host__ __device__ static constexpr int v_piece(int lane, int pair) {
        return D == 128 ? (lane ^ (2 * (pair & 3))) * 16 : (lane ^ (4 * ((pair >> 1) & 1))) * 8;
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
