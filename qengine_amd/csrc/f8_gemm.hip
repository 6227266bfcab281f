// 8-bit products of many rows (f8.hpp): tiles of BT rows x BW weight rows, steps of 128 k through LDS.
//
// LDS holds two stages of activations ([BT][128 bytes], 16-byte chunk c of row r at c ^ (r % 8)), weights (as they lie in
// memory) and the rows' scales of the step, filled by LDS DMA a step ahead. Each MFMA of depth 128 starts from zero and its
// four sums are added at sx sw in fp32.
#include "mfma_tile.hpp"
#include "f8.hpp"

namespace {
using qe_tile::dma16;
using qe_tile::dma4;

__device__ const uint4 kZeros[4] = {};  // what stands behind a row's last column

template <int BT, int BW, int WVT, int WVW, int OUT, bool GROUPED>
__global__ void __launch_bounds__(WVT * WVW * 64) gemm_kernel(F8Mat a, int ntt, int ntw, bool vec) {
    constexpr int NW = WVT * WVW, NTH = NW * 64, TT = BT / WVT / 16, WT = BW / WVW / 16;
    constexpr int kX = BT * 128, kW = BW * 128, kStage = kX + kW + BT * 4;
    constexpr int XD = BT / 8 / NW, WD = BW / 8 / NW;  // DMAs of a wave and step
    static_assert(XD * 8 * NW == BT && WD * 8 * NW == BW && BT / 64 <= NW, "whole DMAs");
    extern __shared__ __align__(16) char lds[];
    const unsigned lds32 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / WVW, ww = wave % WVW, r = lane & 15, g = lane >> 4;
    const int kb = (a.k + 127) >> 7, n16 = (a.n + 15) >> 4;

    // block b runs on XCD b % 8; an XCD takes a run of tiles, in groups of 8 row tiles, so that those on it at a time
    // share their rows and weights in its L2
    const int ntiles = ntt * ntw, per = (ntiles + 7) >> 3, tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || tile >= ntiles) return;
    int tt, tw, e = 0, row0, rows;
    if constexpr (GROUPED) {
        tt = tile / ntw;
        tw = tile % ntw;
        if (!f8_job<NTH>(a.off, a.experts, a.r, BT, tt, reinterpret_cast<int*>(lds), e, row0, rows)) return;
        __syncthreads();
    } else {
        const int full = tile / (8 * ntw), left = min(8, ntt - full * 8), in = tile - full * 8 * ntw;
        tt = full * 8 + in % left;
        tw = in / left;
        row0 = tt * BT;
        rows = min(BT, a.r - row0);
    }
    auto x_row = [&](int i) -> int64_t {  // row i of the tile (the last one again behind it), -1: an index outside x
        const int64_t row = row0 + min(i, rows - 1);
        if (!GROUPED || !a.rows) return row;
        const int at = a.rows[row];
        return (unsigned)at < (unsigned)a.t ? at : -1;
    };
    const char *xp[XD], *wp[WD];
    bool has[XD];
    const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < XD; i++) {
        const int64_t row = x_row((wave * XD + i) * 8 + (lane >> 3));
        has[i] = row >= 0;
        xp[i] = static_cast<const char*>(a.x) + (has[i] ? row : 0) * a.ldx + chunk * 16;
    }
#pragma unroll
    for (int i = 0; i < WD; i++) {
        const int d = wave * WD + i, t16 = min(tw * (BW / 16) + (d >> 1), n16 - 1);
        wp[i] = static_cast<const char*>(a.q) + ((size_t)e * n16 + t16) * kb * 2048 + (d & 1) * 1024 + lane * 16;
    }
    const int64_t srow = wave < BT / 64 ? x_row(wave * 64 + lane) : 0;
    const float* sp = a.xs + (srow < 0 ? 0 : srow) * a.xs_row;
    auto dma_step = [&](int b, int stage) {
        const unsigned to = lds32 + stage * kStage;
        const bool last = b * 128 + 128 > a.k;
#pragma unroll
        for (int i = 0; i < XD; i++) {
            const char* p = xp[i] + (size_t)b * 128;
            if (!has[i] || (last && b * 128 + chunk * 16 >= a.k)) p = reinterpret_cast<const char*>(kZeros);
            dma16(p, to + (wave * XD + i) * 1024);
        }
#pragma unroll
        for (int i = 0; i < WD; i++) dma16(wp[i] + (size_t)b * 2048, to + kX + (wave * WD + i) * 1024);
        if (wave < BT / 64) dma4(srow < 0 ? reinterpret_cast<const float*>(kZeros) : sp + b * a.xs_group, to + kX + kW + wave * 256);
    };
    const int nb = min((tw * BW + ww * WT * 16) >> 7, (a.n - 1) >> 7);
    const float* sw = a.s + ((size_t)e * ((a.n + 127) >> 7) + nb) * kb;
    static_assert(128 % (WT * 16) == 0, "a wave's weight rows lie in one block of 128");

    f32x4_v acc[WT][TT] = {};
    const int xo = (wt * TT * 16 + r) * 128 + ((g ^ (r & 7)) << 4), wo = ww * WT * 2048 + lane * 16;
    dma_step(0, 0);
    for (int b = 0; b < kb; b++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (b + 1 < kb) dma_step(b + 1, (b + 1) & 1);
        const char* x = lds + (b & 1) * kStage;
        const char* w = x + kX;
        const float* sx = reinterpret_cast<const float*>(w + kW);
        const float swb = sw[b];
        i32x8_f8 wf[WT];
#pragma unroll
        for (int i = 0; i < WT; i++)
            wf[i] = f8_join(*reinterpret_cast<const i32x4_f8*>(w + wo + i * 2048), *reinterpret_cast<const i32x4_f8*>(w + wo + i * 2048 + 1024));
#pragma unroll
        for (int t = 0; t < TT; t++) {
            const i32x8_f8 xf = f8_join(*reinterpret_cast<const i32x4_f8*>(x + xo + t * 2048), *reinterpret_cast<const i32x4_f8*>(x + (xo ^ 64) + t * 2048));
            const float s = sx[wt * TT * 16 + t * 16 + r] * swb;
#pragma unroll
            for (int i = 0; i < WT; i++) {
                const f32x4_v p = f8_mfma(wf[i], xf);
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][t][j] = fmaf(p[j], s, acc[i][t][j]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TT; t++) {
        const int row = wt * TT * 16 + t * 16 + r;
        if (row >= rows) continue;
#pragma unroll
        for (int i = 0; i < WT; i++) {
            const int col = tw * BW + (ww * WT + i) * 16 + 4 * g;
            if (col < a.n) f8_store4<OUT>(static_cast<uint16_t*>(a.y) + (int64_t)(row0 + row) * a.ldy, col, a.n, acc[i][t], vec);
        }
    }
}

template <int BT, int BW, int WVT, int WVW, bool GROUPED>
void gemm_t(const F8Mat& a, hipStream_t st) {
    constexpr int kLds = 2 * (BT * 128 + BW * 128 + BT * 4);
    const int64_t ntt = GROUPED ? f8_most_jobs(a.r, a.experts, BT) : (a.r + BT - 1) / BT, ntw = (a.n + BW - 1) / BW;
    CHECK(ntt * ntw <= kF8MaxBlocks, "matmul_f8: %lld row tiles by %lld column tiles are too many for a call", (long long)ntt, (long long)ntw);
    const dim3 grid((unsigned)((ntt * ntw + 7) / 8 * 8)), block(WVT * WVW * 64);
    const bool vec = f8_vec_ok(a.y, a.ldy);
    if (a.out == kF8BF16) gemm_kernel<BT, BW, WVT, WVW, kF8BF16, GROUPED><<<grid, block, kLds, st>>>(a, (int)ntt, (int)ntw, vec);
    else gemm_kernel<BT, BW, WVT, WVW, kF8F16, GROUPED><<<grid, block, kLds, st>>>(a, (int)ntt, (int)ntw, vec);
    HIP_CHECK(hipGetLastError());
}
}  // namespace

void f8_gemm(const F8Mat& a, hipStream_t st) {
    if (a.off) gemm_t<64, 128, 1, 4, true>(a, st);
    else if (a.r <= 64) gemm_t<64, 128, 1, 4, false>(a, st);
    else if (a.r <= 1024) gemm_t<128, 128, 2, 2, false>(a, st);
    else gemm_t<256, 256, 2, 4, false>(a, st);
}

void f8_matmul(const F8Mat& a, hipStream_t st) {
    CHECK(a.n > 0 && a.n <= kF8MaxDim && a.k > 0 && a.k <= kF8MaxDim && a.k % 16 == 0, "matmul_f8: n = %d, k = %d", a.n, a.k);
    CHECK(a.r > 0 && a.r <= kF8MaxRows && a.t >= 0 && a.t <= kF8MaxRows && (a.off || a.t == a.r), "matmul_f8: %d rows of x, %d of y", a.t, a.r);
    CHECK(a.experts > 0 && a.experts <= kF8MaxExperts && (a.off || (a.experts == 1 && !a.rows)), "matmul_f8: %d matrices", a.experts);
    CHECK(a.q && a.s && a.y && (a.t == 0 || (a.x && a.xs)), "matmul_f8: a tensor is missing");
    CHECK(((uintptr_t)a.q & 15) == 0 && ((uintptr_t)a.x & 15) == 0 && a.ldx % 16 == 0, "matmul_f8: x and its rows are 16-byte aligned");
    const bool few = a.off ? a.r <= (int64_t)a.experts * 8 : a.r <= 32;
    if (few) f8_dec(a, st);
    else f8_gemm(a, st);
}
