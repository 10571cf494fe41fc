// The 4-bit paged key/value cache shared by its store, load and attention kernels.
//
// The cache is [pages, heads, page_size / 16] records, one for every 16 tokens of a head, so one
// contiguous 16-byte aligned copy brings a whole attention tile.  A record of head size D
// (N = D / 64 groups a row) holds 18 D bytes:
//
//   key codes    16 rows of D / 2 bytes   element 64 G + 16 t + 8 h + n: byte t 8N + 8 G + 4 h + n / 2
//   value codes  16 rows of D / 2 bytes   element 64 G + 8 c + n:        byte (c ^ 4 ((row >> 1) & 1)) 4N + 4 G + n / 2
//   key (scale, minimum) pairs in bf16    [16 rows][N]
//   value pairs                           [16 rows][N]
//
// the even n in a byte's low half.  A code q in 0..15 stands for minimum + scale q.  The orders
// are those in which the attention kernel's lanes take a row: its MMA sums over a head's elements
// in any order, so a lane's share of a row is contiguous (one 16-byte shared-memory read for keys,
// one 8-byte read for values at D = 128), and the value chunks of rows 2 and 3 of every four change
// places so that the four rows a half-warp reads fall in different banks.
//
// Quantisation of a group of 64: minimum = bf16(min x), scale = bf16((max x - min x) / 15),
// q = rint((x - minimum) / scale) clamped to 0..15 (0 when the scale is 0).  bf16 keeps the range of
// both 16-bit types; the codes are taken against the rounded pair, so its rounding costs at most
// the clamped ends.  Differences and quotients are IEEE fp32 operations, each rounded: an element that fp32 does
// not tell from a tie between two codes goes where the tie goes.  A group whose values or range are not finite is stored with minimum NaN.
#pragma once

#include "sf_common.cuh"
#include "sm100.cuh"

namespace kv4 {

template <int NG>
struct Record {
    static constexpr int D = 64 * NG;
    static constexpr int ROW = 32 * NG;           // bytes of one row's codes
    static constexpr int K = 0;
    static constexpr int V = 16 * ROW;
    static constexpr int KP = 32 * ROW;           // key (scale, minimum) pairs, 4 NG bytes a row
    static constexpr int VP = KP + 64 * NG;
    static constexpr int BYTES = VP + 64 * NG;    // 18 D
};

// Status codes and places reported through sf_kernel_status (code 3: an index out of range).
constexpr unsigned BAD_INDEX = 3;
constexpr unsigned AT_STORE_SLOT = 110, AT_LOAD_SLOT = 111, AT_PAGE = 112, AT_LENGTH = 113, AT_WAIT = 114;

__device__ __forceinline__ void report(sm100::KernelStatus* st, unsigned code, unsigned where) {
    if (atomicCAS(&st->code, 0u, code) == 0u) st->where = where;
}

// Read and clear a pair of status words (a `__device__` array of two); the wait's word comes first.
template <typename W>
int read_status(W& words, uint32_t* code, uint32_t* where, cudaStream_t stream) {
    sm100::KernelStatus h[2] = {{0, 0}, {0, 0}};
    if (cudaMemcpyFromSymbolAsync(h, words, sizeof(h), 0, cudaMemcpyDeviceToHost, stream) != cudaSuccess) return SF_EDEVICE;
    if (cudaStreamSynchronize(stream) != cudaSuccess) return SF_EDEVICE;
    if (h[0].code || h[1].code) {
        const sm100::KernelStatus zero[2] = {{0, 0}, {0, 0}};
        cudaMemcpyToSymbolAsync(words, zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream);
        cudaStreamSynchronize(stream);
    }
    const sm100::KernelStatus& first = h[1].code ? h[1] : h[0];
    *code = first.code;
    *where = first.where;
    return SF_OK;
}

}  // namespace kv4
