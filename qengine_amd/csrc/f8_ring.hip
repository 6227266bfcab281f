// 8-bit products whose weights are read for few rows each (f8.hpp): BT rows x BW weight rows a block, four waves with all rows
// x BW / 4 of it each, in steps of 128 k. Bound by the weights' bytes: both operands come by LDS DMA into a ring of S stages, so that S - 1 steps are
// on their way without a register. Two more waves do nothing but issue the DMAs: a step's 28 (BT 64, BW 128) take the address unit 450
// cycles, as long as its products, and the waves that multiplied stood behind their own (1 block a CU: 1570 cycles a step).
#include "f8_tile.hpp"

namespace {
template <int BT, int BW, int S>
constexpr int ring_stage() { return BT * 128 + BW * 128 + (BT < 64 ? 64 : BT) * 4 + 256; }

constexpr int kIssue = 2, kThreads = (4 + kIssue) * 64;  // waves that issue DMAs

template <int BT, int BW, int S, int OUT, bool GROUPED>
__global__ void __launch_bounds__(kThreads) ring_kernel(F8Mat a, F8Split sp, int ntt, int ntw, bool vec) {
    constexpr int TT = BT / 16, WT = BW / 64, SW = (BT + 63) / 64;
    constexpr int XD = BT / 8 / kIssue, WD = BW / 8 / kIssue, NDMA = XD + WD + (SW + 1 + kIssue - 1) / kIssue;  // DMAs of an issuing wave and step
    constexpr int kStage = ring_stage<BT, BW, S>(), kX = BT * 128, oS = kX + BW * 128, oW = oS + (BT < 64 ? 64 : BT) * 4;
    constexpr int kLeft = (S - 2) * NDMA;
    static_assert(kLeft < 64 && BT % (8 * kIssue) == 0 && BW % 64 == 0, "vmcnt counts to 63; whole DMAs");
    extern __shared__ __align__(16) char lds[];
    const unsigned lds32 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int blocks = (a.k + 127) >> 7, n16 = (a.n + 15) >> 4;

    int item, tt = 0, tw, e = 0, row0, rows, z = 0;
    if constexpr (GROUPED) {
        const int idx = blockIdx.x >> 3;
        tw = idx % ntw;
        if (!f8_job<kThreads>(a.off, a.experts, a.r, BT, blockIdx.x & 7, 8, idx / ntw, reinterpret_cast<int*>(lds), e, row0, rows)) return;
        __syncthreads();
    } else {
        if (!xcd_item(ntt * ntw * sp.parts, item)) return;
        z = item / (ntt * ntw);
        tile_place(item % (ntt * ntw), ntt, ntw, tt, tw);
        row0 = tt * BT;
        rows = min(BT, a.r - row0);
    }
    const int from = GROUPED ? 0 : (int)((int64_t)blocks * z / sp.parts), kb = GROUPED ? blocks : (int)((int64_t)blocks * (z + 1) / sp.parts) - from;

    if (wave >= 4) {
        const int part = wave - 4;
        // row i of the tile (the last one again behind it) in x; an index outside x: row 0, and zeros in y
        auto x_row = [&](int i) -> int64_t {
            const int64_t row = row0 + min(i, rows - 1);
            if (!GROUPED || !a.rows) return row;
            const int at = a.rows[row];
            return (unsigned)at < (unsigned)a.t ? at : 0;
        };
        // chunks behind k take the block's first: a row's own finite values times the weights' zeros there
        const int chunk = (lane & 7) ^ (lane >> 3), back = chunk * 16 < a.k - (blocks - 1) * 128 ? 0 : -chunk * 16, tail = blocks - 1 - from;
        const char* xp[XD];
#pragma unroll
        for (int i = 0; i < XD; i++)
            xp[i] = static_cast<const char*>(a.x) + x_row((part * XD + i) * 8 + (lane >> 3)) * a.ldx + chunk * 16 + (int64_t)from * 128;
        // weights from a base that moves by a step, and this lane's offsets of the tile (rows behind n: the last ones again)
        // (n and k are below 2^20 + 1: the offsets within a tile stay below 2^32)
        const char* wb = scalar(static_cast<const char*>(a.q) + (((size_t)e * n16 + tw * (BW / 16)) * blocks + from) * 2048);
        uint32_t wi[WD];
#pragma unroll
        for (int i = 0; i < WD; i++) {
            const int d = part * WD + i;
            wi[i] = (uint32_t)min(d >> 1, n16 - 1 - tw * (BW / 16)) * (uint32_t)(blocks * 2048) + (d & 1) * 1024 + lane * 16;
        }
        // scales: DMA j of the step's SW + 1 is 64 rows', the last one (and what fills up the count) the weights' blocks of 128 rows'
        constexpr int SD = NDMA - XD - WD;
        const float* sw = a.s + ((size_t)e * ((a.n + 127) >> 7) + min((tw * BW >> 7) + (lane & 3), (a.n - 1) >> 7)) * blocks + from;
        const float* sc[SD];
#pragma unroll
        for (int i = 0; i < SD; i++) sc[i] = a.xs + (part * SD + i < SW ? x_row((part * SD + i) * 64 + lane) * a.xs_row : 0) + from * a.xs_group;
        int f_b = 0, f_stage = 0;  // the next step that is fetched, and its stage
        auto fetch = [&] {
            const unsigned to = lds32 + f_stage * kStage;
#pragma unroll
            for (int i = 0; i < WD; i++) dma16_at(wb, wi[i], to + kX + (part * WD + i) * 1024);
            if (f_b == tail) {
#pragma unroll
                for (int i = 0; i < XD; i++) dma16(xp[i] + back, to + (part * XD + i) * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < XD; i++) dma16(xp[i], to + (part * XD + i) * 1024);
            }
#pragma unroll
            for (int i = 0; i < SD; i++) {
                const int j = part * SD + i;
                dma4(j < SW ? sc[i] : sw, to + (j < SW ? oS + j * 256 : oW));
                sc[i] += a.xs_group;
            }
            sw++;
            wb = scalar(wb + 2048);
#pragma unroll
            for (int i = 0; i < XD; i++) xp[i] += 128;
            if (++f_stage == S) f_stage = 0;
            f_b++;
        };
        for (int i = 0; i < S - 1 && i < kb; i++) fetch();
        for (int i = 0; i < kb; i++) {
            // the step's DMAs are there (with fewer than S - 2 steps behind it all are waited for); the waves that multiply have read
            // the step before, whose stage is the next one filled
            if (f_b < kb) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kLeft) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (f_b < kb) fetch();
        }
        return;
    }

    f32x4_v acc[WT][TT] = {};
    const int xo = r * 128 + ((g ^ (r & 7)) << 4);
    int stage = 0;
    for (int b = 0; b < kb; b++) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const char* p = lds + stage * kStage;
        i32x8_f8 w[WT];
#pragma unroll
        for (int i = 0; i < WT; i++) {
            const char* q = p + kX + (wave * WT + i) * 2048 + lane * 16;
            w[i] = f8_join(*reinterpret_cast<const i32x4_f8*>(q), *reinterpret_cast<const i32x4_f8*>(q + 1024));
        }
        float sw[WT];  // of its 16 rows: BW = 192 has waves on both sides of a block's end
#pragma unroll
        for (int i = 0; i < WT; i++) sw[i] = *reinterpret_cast<const float*>(p + oW + ((tw * (BW / 16) + wave * WT + i) / 8 - (tw * BW >> 7)) * 4);
#pragma unroll
        for (int t = 0; t < TT; t++) {
            const i32x8_f8 x = f8_join(*reinterpret_cast<const i32x4_f8*>(p + xo + t * 2048), *reinterpret_cast<const i32x4_f8*>(p + (xo ^ 64) + t * 2048));
            const float s = *reinterpret_cast<const float*>(p + oS + (t * 16 + r) * 4);
#pragma unroll
            for (int i = 0; i < WT; i++) {
                const f32x4_v v = f8_mfma(w[i], x);
                const float f = s * sw[i];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][t][j] = fmaf(v[j], f, acc[i][t][j]);
            }
        }
        if (++stage == S) stage = 0;
    }
    const int col = (tw * (BW / 16) + wave * WT) * 16;
    if (!GROUPED && sp.parts > 1) {
        f32x4_v* const to = sp.sums + ((((size_t)tt * ntw + tw) * sp.parts + z) * 4 + wave) * TT * WT * 64 + lane;
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < WT; i++) to[(t * WT + i) * 64] = acc[i][t];
    } else if (col < a.n) {
        char* const out = lds + S * kStage + wave * 16 * WT * 32;  // 16 rows at a time
#pragma unroll
        for (int t = 0; t < TT; t++) {
            f32x4_v v[WT][1];
#pragma unroll
            for (int i = 0; i < WT; i++) v[i][0] = acc[i][t];
            store_wave<1, WT, OUT>(v, out, lane, static_cast<uint16_t*>(a.y) + (int64_t)(row0 + t * 16) * a.ldy + col, a.ldy, rows - t * 16, a.n - col, vec,
                                   [&](int i) { return GROUPED && a.rows && (unsigned)a.rows[row0 + t * 16 + i] >= (unsigned)a.t; });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

template <int BT, int BW, int S, bool GROUPED>
void ring_t(const F8Mat& a, int parts, hipStream_t st) {
    constexpr int kLds = S * ring_stage<BT, BW, S>() + BW * 32;
    static_assert(kLds <= 160 * 1024, "LDS of a CU");
    const int64_t ntt = GROUPED ? f8_most_jobs(a.r, a.experts, BT) : (a.r + BT - 1) / BT, ntw = (a.n + BW - 1) / BW;
    CHECK(ntt * ntw * parts <= kF8MaxBlocks, "matmul_f8: %lld row tiles by %lld column tiles are too many for a call", (long long)ntt, (long long)ntw);
    const bool vec = a.ldy % 8 == 0 && ((uintptr_t)a.y & 15) == 0;
    auto run = [&](const F8Split& sp) {
        const dim3 grid(GROUPED ? xcd_blocks(ntt) * (unsigned)ntw : xcd_blocks(ntt * ntw * sp.parts)), block(kThreads);
        if (a.out == kF8BF16) ring_kernel<BT, BW, S, kF8BF16, GROUPED><<<grid, block, kLds, st>>>(a, sp, (int)ntt, (int)ntw, vec);
        else ring_kernel<BT, BW, S, kF8F16, GROUPED><<<grid, block, kLds, st>>>(a, sp, (int)ntt, (int)ntw, vec);
        HIP_CHECK(hipGetLastError());
    };
    if constexpr (GROUPED) {
        run({});
    } else {
        if (parts < 2) return run({});
        WsHold hold(st);
        const F8Split sp = f8_split(hold, ntt * ntw, parts, BT, BW);
        run(sp);
        if (sp.parts < 2) return;
        const dim3 grid((unsigned)(ntt * ntw * 4 * (BT / 16)));
        if (a.out == kF8BF16) sum_kernel<BT, BW, 1, 4, 1, kF8BF16><<<grid, dim3(64), 0, st>>>(a, sp, (int)ntw, vec);
        else sum_kernel<BT, BW, 1, 4, 1, kF8F16><<<grid, dim3(64), 0, st>>>(a, sp, (int)ntw, vec);
        HIP_CHECK(hipGetLastError());
    }
}
}  // namespace

// Stages: three keep a block fed (four or six took the same time or longer); two where a third would leave one block a CU.
void f8_ring(const F8Mat& a, int bt, int bw, int parts, hipStream_t st) {
    if (a.off) {
        if (bt == 64) ring_t<64, 128, 3, true>(a, 1, st);
        else ring_t<128, 128, 2, true>(a, 1, st);
    } else if (bt == 32) {
        if (bw == 64) ring_t<32, 64, 4, false>(a, parts, st);
        else if (bw == 128) ring_t<32, 128, 3, false>(a, parts, st);
        else ring_t<32, 192, 3, false>(a, parts, st);
    } else if (bt == 64) {
        if (bw == 64) ring_t<64, 64, 4, false>(a, parts, st);
        else if (bw == 128) ring_t<64, 128, 3, false>(a, parts, st);
        else ring_t<64, 192, 3, false>(a, parts, st);
    } else {
        if (bw == 64) ring_t<128, 64, 3, false>(a, parts, st);
        else if (bw == 128) ring_t<128, 128, 2, false>(a, parts, st);
        else ring_t<128, 192, 3, false>(a, parts, st);
    }
}
