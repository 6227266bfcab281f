// What the tile kernels of 8-bit products share (f8_gemm.hip, f8_ring.hip): where a tile lies, and its way out.
#pragma once
#include "f8.hpp"
#include "mfma_tile.hpp"

namespace {
using qe_tile::dma16;
using qe_tile::dma16_at;
using qe_tile::dma4;
using qe_tile::dma4_at;

// the same address in scalar registers, where a DMA takes its base from
__device__ __forceinline__ const char* scalar(const char* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const char*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 |
                                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
}

// K split (one matrix): a tile's 128-k blocks in `parts` ranges, whose sums go to memory as the lanes hold them and are added in
// the order of the ranges by sum_kernel
struct F8Split {
    f32x4_v* sums = nullptr;  // [row tile][column tile][range][wave][product][lane]
    int parts = 1;
};

// Block b runs on XCD b % 8; an XCD takes a run of the items (tiles, or ranges outermost), so that those on it at a time share
// rows and weights in its L2: tiles in groups of 8 row tiles, inside a group row tiles innermost. Grouped: a run of the segments' blocks
// of rows, as many as there are (shared out by the most there can be, two XCDs of eight had nothing to do: 320 us for 40960
// rows of 512 experts, 1024 x 2048).
__device__ __forceinline__ bool xcd_item(int items, int& item) {
    const int per = (items + 7) >> 3;
    item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    return (int)(blockIdx.x >> 3) < per && item < items;
}
__device__ __forceinline__ void tile_place(int tile, int ntt, int ntw, int& tt, int& tw) {
    const int full = tile / (8 * ntw), left = min(8, ntt - full * 8), in = tile - full * 8 * ntw;
    tt = full * 8 + in % left;
    tw = in / left;
}
inline unsigned xcd_blocks(int64_t items) { return (unsigned)((items + 7) / 8 * 8); }

// A wave's sums to rows of y through its part of LDS, NT tokens x 16 of WT x 16 columns: stored as they lie (8 bytes of 16 rows a store)
// a tile of 256 x 256 took 7 us, read back as 16-byte pieces of whole rows 2. Chunk c of row i lies at c ^ (i % C).
// y: the wave's first row and column; rows, cols: how many of them there are; bad(i): row i is zeros
template <int TT, int WT, int OUT, class Bad>
__device__ __forceinline__ void store_wave(const f32x4_v (&acc)[WT][TT], char* out, int lane, uint16_t* y, int64_t ldy, int rows, int cols, bool vec, Bad bad) {
    constexpr int C = WT * 2, M = (C & (C - 1)) == 0 ? C - 1 : 0;  // 16-byte chunks of a row (six of them stay in order)
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < WT; i++) {
            const f32x4_v v = acc[i][t];
            *reinterpret_cast<uint2*>(out + ((t * 16 + r) * C + ((2 * i + (g >> 1)) ^ (r & M))) * 16 + (g & 1) * 8) =
                OUT == kF8BF16 ? uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])} : uint2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
    for (int j = 0; j < (TT * C + 3) / 4; j++) {
        const int at = j * 64 + lane, i = at / C, c = at % C;
        if (at >= TT * 16 * C || i >= rows || c * 8 >= cols) continue;
        uint4 v = *reinterpret_cast<const uint4*>(out + (i * C + (c ^ (i & M))) * 16);
        if (bad(i)) v = uint4{0, 0, 0, 0};
        uint16_t* const to = y + i * ldy + c * 8;
        if (vec && c * 8 + 8 <= cols) {
            *reinterpret_cast<uint4*>(to) = v;
        } else {
            const uint32_t pairs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (c * 8 + k < cols) to[k] = (uint16_t)(pairs[k >> 1] >> (16 * (k & 1)));
        }
    }
}

// the sums of a split tile's ranges: a wave takes QT of the TT x 16 rows of one wave of the tile
template <int BT, int BW, int WVT, int WVW, int QT, int OUT>
__global__ void __launch_bounds__(64) sum_kernel(F8Mat a, F8Split sp, int ntw, bool vec) {
    constexpr int NW = WVT * WVW, TT = BT / WVT / 16, WT = BW / WVW / 16, Q = TT / QT;
    __shared__ __align__(16) char out[QT * 16 * WT * 32];
    const int lane = threadIdx.x, q = blockIdx.x % Q, wave = blockIdx.x / Q % NW, tile = blockIdx.x / Q / NW;
    const int tt = tile / ntw, tw = tile % ntw;
    const int first = tt * BT + wave / WVW * TT * 16 + q * QT * 16, col = tw * BW + wave % WVW * WT * 16;
    if (first >= a.r || col >= a.n) return;
    f32x4_v acc[WT][QT] = {};
    for (int z = 0; z < sp.parts; z++) {
        const f32x4_v* p = sp.sums + ((((size_t)tile * sp.parts + z) * NW + wave) * TT + q * QT) * WT * 64 + lane;
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
            for (int i = 0; i < WT; i++) {
                const f32x4_v v = p[(t * WT + i) * 64];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][t][j] += v[j];
            }
    }
    store_wave<QT, WT, OUT>(acc, out, lane, static_cast<uint16_t*>(a.y) + (int64_t)first * a.ldy + col, a.ldy, a.r - first, a.n - col, vec,
                            [](int) { return false; });
}

// room for the sums of tiles * parts blocks of BT x BW: a stream's buffer holds a block of 256 x 256 for each CU (64 MB) from its first split
// on, so that it never grows (f8_matmul.cpp splits where the blocks are no more than the CUs); a graph's what its calls need. No split where
// they need more, or without memory.
inline F8Split f8_split(WsHold& hold, int64_t tiles, int parts, int bt, int bw) {
    F8Split sp;
    const size_t whole = (size_t)qe_num_cus() * 256 * 256 * 4, bytes = (size_t)tiles * parts * bt * bw * 4;
    if (parts < 2 || bytes > whole) return sp;
    sp.sums = static_cast<f32x4_v*>(hold.get(kWsF8, bytes, false, whole));
    if (sp.sums) sp.parts = parts;
    return sp;
}
}  // namespace
