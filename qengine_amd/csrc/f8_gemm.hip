// 8-bit products of many rows (f8.hpp): tiles of BT rows x BW weight rows in steps of 128 k.
//
// A wave holds TT x WT tiles of 16 x 16 sums. Both operands go through LDS, filled by LDS DMA. What a step begins with is there a
// step early, so that no wave waits for LDS behind the barrier: weights are read into registers a step ahead, and the first 16 rows
// of each wave and the rows' scales have rings of three. Each MFMA of depth 128 starts from zero; its four sums are added at sx sw
// in fp32 behind the next ones.
// Bound by the matrix cores and what keeps them waiting: a step of 256 x 256 has 2048 cycles of products a SIMD. Issued at once its
// DMAs kept the waves at the address unit (64 bytes a cycle, 1000 to 1500 cycles) ahead of the products: 4490 cycles a step; the rows' and
// scales' in its first half, the weights', which have until the middle of the next step, in its second: about 3200. 8192 rows of 17408 x
// 5120: 633 to 654 us, 2.23 to 2.31 PFLOP/s, 1.6 us a step and round; with no DMA in the loop 1.15, with zeros for data (no power limit) 13 % less in all. Two
// barriers a step: in its middle (the weights of the step before have come) and at its end. Not faster (against
// 652): DMAs closer together or further apart (651 to 672), a third stage of rows (664), weights straight into registers (765: two waves fetch the same ones).
#include "f8_tile.hpp"
#include <type_traits>

namespace {
template <int BT, int BW, int WVT, int WVW, int OUT, bool GROUPED>
__global__ void __launch_bounds__(WVT * WVW * 64, 2) gemm_kernel(F8Mat a, F8Split sp, int ntt, int ntw, bool vec) {
    constexpr int NW = WVT * WVW, NTH = NW * 64, TT = BT / WVT / 16, WT = BW / WVW / 16;
    constexpr int kX = BT * 128, kW = BW * 128, kFirst = WVT * 2048, kS = BT * 4 + 256;  // bytes of a stage
    constexpr int oW = 2 * kX, oFirst = oW + 2 * kW, oS = oFirst + 3 * kFirst;
    constexpr int XD = BT / 8 / NW, WD = BW / 8 / NW;  // DMAs of a wave and step
    static_assert(XD * 8 * NW == BT && WD * 8 * NW == BW && BT / 64 < NW && TT % 2 == 0 && BW % 128 == 0, "whole DMAs");
    static_assert(128 % (WT * 16) == 0, "a wave's weight rows lie in one block of 128");
    extern __shared__ __align__(16) char lds[];
    const unsigned lds32 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wave / WVW, ww = wave % WVW, r = lane & 15, g = lane >> 4;
    const int blocks = (a.k + 127) >> 7, n16 = (a.n + 15) >> 4;  // of 128 k

    int item, tt = 0, tw, e = 0, row0, rows, z = 0;
    if constexpr (GROUPED) {
        const int idx = blockIdx.x >> 3;
        tw = idx % ntw;
        if (!f8_job<NTH>(a.off, a.experts, a.r, BT, blockIdx.x & 7, 8, idx / ntw, reinterpret_cast<int*>(lds), e, row0, rows)) return;
        __syncthreads();
    } else {
        if (!xcd_item(ntt * ntw * sp.parts, item)) return;
        z = item / (ntt * ntw);
        tile_place(item % (ntt * ntw), ntt, ntw, tt, tw);
        row0 = tt * BT;
        rows = min(BT, a.r - row0);
    }
    const int from = (int)((int64_t)blocks * z / sp.parts), kb = (int)((int64_t)blocks * (z + 1) / sp.parts) - from;  // this range
    // chunks behind k take the block's first: a row's own finite values times the weights' zeros there
    const int chunk = (lane & 7) ^ (lane >> 3), back = chunk * 16 < a.k - (blocks - 1) * 128 ? 0 : -chunk * 16;
    // Rows of x by 32-bit offsets, from the tile's first (rows are less than 2^24 bytes apart, their scales less than 2^22 elements), or by
    // index from the first of all (x and its scales are then less than 2^32 bytes). Behind the last row that one again.
    const bool by_index = GROUPED && a.rows;
    auto x_row = [&](int i) -> uint32_t {
        i = min(i, rows - 1);
        if (!by_index) return i;
        const uint32_t at = a.rows[row0 + i];
        return at < (uint32_t)a.t ? at : 0;  // an index outside x: row 0, and zeros in y
    };
    const int64_t x_first = by_index ? 0 : row0;
    const char* const x0 = static_cast<const char*>(a.x) + x_first * a.ldx + (int64_t)from * 128;
    uint32_t xi[XD];
#pragma unroll
    for (int i = 0; i < XD; i++) xi[i] = x_row((wave * XD + i) * 8 + (lane >> 3)) * (uint32_t)a.ldx + chunk * 16;
    // scales of the rows, 64 a wave, and of the tile's blocks of 128 weight rows, by the wave after them
    const char* s0p = reinterpret_cast<const char*>(a.xs + x_first * a.xs_row + from * a.xs_group);
    int64_t s_next = a.xs_group * 4;
    uint32_t si = wave < BT / 64 ? x_row(wave * 64 + lane) * (uint32_t)(a.xs_row * 4) : 0;
    if (wave >= BT / 64) {  // (the waves after it fetch the same again, so that all count the same DMAs)
        s0p = reinterpret_cast<const char*>(a.s + (size_t)e * ((a.n + 127) >> 7) * blocks + from);
        s_next = 4;
        si = (uint32_t)min(tw * (BW / 128) + (lane & (BW / 128 - 1)), (a.n - 1) >> 7) * (uint32_t)(blocks * 4);
    }
    const int t16 = tw * (BW / 16) + ww * WT;  // the wave's first 16 weight rows
    const char* const w0 = static_cast<const char*>(a.q) + (((size_t)e * n16 + tw * (BW / 16)) * blocks + from) * 2048;
    // DMAs of this wave, past the last block that block again (nobody reads it): 8 rows of x, block b, to LDS byte `to`
    const int tail = blocks - 1 - from;  // the matrix's last block
    uint32_t wi[WD];                     // (uniform) bytes from the first tile's first block: n and k below 2^20 + 1, 16 tiles: below 2^32
#pragma unroll
    for (int i = 0; i < WD; i++) {
        const int d = wave * WD + i;
        wi[i] = (uint32_t)min(d >> 1, n16 - 1 - tw * (BW / 16)) * (uint32_t)(blocks * 2048) + (d & 1) * 1024;
    }
    auto dma_x = [&](int i, int b, unsigned to) {
        b = min(b, kb - 1);
        dma16_at(scalar(x0 + b * 128), xi[i] + (b == tail ? back : 0), to);
    };
    auto dma_w = [&](int i, int b, unsigned to) {
        dma16_at(scalar(w0 + (size_t)min(b, kb - 1) * 2048 + wi[i]), lane * 16, to + (wave * WD + i) * 1024);
    };
    auto dma_s = [&](int b, unsigned to) {
        dma4_at(scalar(s0p + min(b, kb - 1) * s_next), si, to + min(wave, BT / 64) * 256);
    };
    // the same for DMA number i of a wave's rows: their first 16 go to the ring for block `early`, the others to a stage
    auto dma_rows = [&](int i, int b, unsigned to, int early, unsigned ring) {
        const int d = wave * XD + i, f = d % (2 * TT);
        dma_x(i, f < 2 ? early : b, f < 2 ? ring + (d / (2 * TT) * 2 + f) * 1024 : to + d * 1024);
    };

    // The sums of product number p = t WT + i wait in a ring while the next two products are under way; the step before's last two
    // are added before the first two of a step take their places
    constexpr int RING = 3, LAG = RING - 1, NP = TT * WT, H = NP / 2, EV = H / (XD + 1), RW = H / (2 * WT);
    static_assert((NP - LAG) % RING == 0 && WT > LAG, "the last sums lie where the first ones go; scales outlast their sums");
    static_assert(EV > 0 && WD <= XD + 1 && RW > 0, "a step's DMAs and reads find a product");
    f32x4_v acc[WT][TT] = {}, part[RING] = {};
    i32x8_f8 w[2][WT];
    i32x8_f8 x[2];
    float sc[TT] = {};  // scales of the step's rows; the last two's of the step before until their turn
    const int xo = r * 128 + ((g ^ (r & 7)) << 4), so = (wt * TT * 16 + r) * 4;
    auto load_w = [&](int to, int i, int h, const char* p) {  // half h of tile i
        const i32x4_f8 v = *reinterpret_cast<const i32x4_f8*>(p + (ww * WT + i) * 2048 + h * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) w[to][i][h * 4 + j] = v[j];
    };
    auto load_x = [&](int to, const char* p) {  // p: 16 rows
        x[to] = f8_join(*reinterpret_cast<const i32x4_f8*>(p + xo), *reinterpret_cast<const i32x4_f8*>(p + (xo ^ 64)));
    };
    auto load_s = [&](const char* p, int t) { return *reinterpret_cast<const float*>(p + so + t * 64); };
    auto load_sw = [&](const char* p) { return *reinterpret_cast<const float*>(p + BT * 4 + (ww * WT >> 3) * 4); };
    auto arrive = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    auto flush = [&](int p) {
        const int i = p % WT, t = p / WT;
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][t][j] = fmaf(part[p % RING][j], sc[t], acc[i][t][j]);
        asm volatile("" : "+v"(acc[i][t]));  // here, not behind the step's branches, where the compiler sinks it
    };
#pragma unroll
    for (int i = 0; i < XD; i++) {
        dma_rows(i, 0, lds32, 0, lds32 + oFirst);
        if ((wave * XD + i) % (2 * TT) < 2) dma_rows(i, 0, 0, 1, lds32 + oFirst + kFirst);
    }
#pragma unroll
    for (int i = 0; i < WD; i++) {
        dma_w(i, 0, lds32 + oW);
        dma_w(i, 1, lds32 + oW + kW);
    }
    dma_s(0, lds32 + oS);
    dma_s(1, lds32 + oS + kS);
    arrive();
    int ring = 0;
#pragma unroll
    for (int i = 0; i < 2 * WT; i++) load_w(0, i / 2, i % 2, lds + oW);
    load_x(0, lds + oFirst + wt * 2048);
    float s0 = load_s(lds + oS, 0), sw0 = load_sw(lds + oS);
    arrive();  // the first weights are read: their stage is free
    // Step b, c = b % 2: products of weights w[c] and rows in stage c and in the ring; reads weights b + 1 from stage 1 - c; fetches
    // rows b + 1 to stage 1 - c, weights b + 2 to stage c, first rows and scales b + 2 to the ring
    auto step = [&](int b, auto c) {
        constexpr int cur = decltype(c)::value;
        const int next = ring == 2 ? 0 : ring + 1, after = next == 2 ? 0 : next + 1;
        const float swb = sw0;
        float s = s0;
#pragma unroll
        for (int t = 0; t < TT; t++) {
            sc[t] = s * swb;
#pragma unroll
            for (int i = 0; i < WT; i++) {
                const int p = t * WT + i;
                if (p < LAG) flush(NP - LAG + p);
                part[p % RING] = f8_mfma(w[cur][i], x[t & 1]);
                if (i == 0) {  // behind the product that needs what was read before: ahead of it the compiler waits for both
                    __builtin_amdgcn_sched_barrier(0);
                    if (t + 1 < TT) {
                        load_x((t + 1) & 1, lds + cur * kX + (wt * TT + t + 1) * 2048);
                        s = load_s(lds + oS + ring * kS, t + 1);
                    } else {
                        load_x(0, lds + oFirst + next * kFirst + wt * 2048);
                        s0 = load_s(lds + oS + next * kS, 0);
                        sw0 = load_sw(lds + oS + next * kS);
                    }
                }
                if (p >= LAG) flush(p - LAG);
                if (p < H && p % EV == 0) {
                    const int j = p / EV;
                    if (j < XD) dma_rows(j, b + 1, lds32 + (cur ^ 1) * kX, b + 2, lds32 + oFirst + after * kFirst);
                    else if (j == XD) dma_s(b + 2, lds32 + oS + after * kS);
                } else if (p >= H && (p - H) % EV == 0) {
                    if ((p - H) / EV < WD) dma_w((p - H) / EV, b + 2, lds32 + oW + cur * kW);
                }
                if (p >= H && (p - H) % RW == RW - 1) load_w(cur ^ 1, (p - H) / RW / 2, (p - H) / RW % 2, lds + oW + (cur ^ 1) * kW);
                // the weights fetched in the step before are there, of all waves
                if (p == H - 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(XD + 1) : "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        ring = next;
        // what the next step begins with is read (the compiler learns it here: it would wait again behind the barrier)
        asm volatile("" : "+v"(x[0]), "+v"(s0), "+v"(sw0));
#pragma unroll
        for (int i = 0; i < WT; i++) asm volatile("" : "+v"(w[cur ^ 1][i]));
        // the rows and scales fetched in this step are there (the weights have until the middle of the next), and all have read their stages
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WD) : "memory");
    };
    int b = 0;
    for (; b + 2 <= kb; b += 2) {
        step(b, std::integral_constant<int, 0>{});
        step(b + 1, std::integral_constant<int, 1>{});
    }
    if (b < kb) step(b, std::integral_constant<int, 0>{});
#pragma unroll
    for (int p = NP - LAG; p < NP; p++) flush(p);
    arrive();  // nothing is on its way to LDS any more
    const int first = wt * TT * 16;  // row of the tile
    if (!GROUPED && sp.parts > 1) {
        f32x4_v* const to = sp.sums + ((((size_t)tt * ntw + tw) * sp.parts + z) * NW + wave) * NP * 64 + lane;
#pragma unroll
        for (int p = 0; p < NP; p++) to[p * 64] = acc[p % WT][p / WT];
        return;
    }
    // through the stages' LDS, which the last barrier freed
    static_assert(NW * TT * 16 * WT * 32 <= 2 * (kX + kW), "every wave's rows fit the stages");
    if (first < rows && t16 * 16 < a.n)
        store_wave<TT, WT, OUT>(acc, lds + wave * TT * 16 * WT * 32, lane, static_cast<uint16_t*>(a.y) + (int64_t)(row0 + first) * a.ldy + t16 * 16,
                                a.ldy, rows - first, a.n - t16 * 16, vec,
                                [&](int i) { return by_index && (unsigned)a.rows[row0 + first + i] >= (unsigned)a.t; });
}

template <int BT, int BW, int WVT, int WVW, bool GROUPED>
void gemm_t(const F8Mat& a, int parts, hipStream_t st) {
    constexpr int kLds = 2 * 128 * (BT + BW) + 3 * (WVT * 2048 + BT * 4 + 256);
    const int64_t ntt = GROUPED ? f8_most_jobs(a.r, a.experts, BT) : (a.r + BT - 1) / BT, ntw = (a.n + BW - 1) / BW;
    CHECK(ntt * ntw * parts <= kF8MaxBlocks, "matmul_f8: %lld row tiles by %lld column tiles are too many for a call", (long long)ntt, (long long)ntw);
    const bool vec = a.ldy % 8 == 0 && ((uintptr_t)a.y & 15) == 0;
    auto run = [&](const F8Split& sp) {
        const dim3 grid(GROUPED ? xcd_blocks(ntt) * (unsigned)ntw : xcd_blocks(ntt * ntw * sp.parts)), block(WVT * WVW * 64);
        if (a.out == kF8BF16) gemm_kernel<BT, BW, WVT, WVW, kF8BF16, GROUPED><<<grid, block, kLds, st>>>(a, sp, (int)ntt, (int)ntw, vec);
        else gemm_kernel<BT, BW, WVT, WVW, kF8F16, GROUPED><<<grid, block, kLds, st>>>(a, sp, (int)ntt, (int)ntw, vec);
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
        constexpr int QT = 2;  // of a wave's eight 16-row tiles a block of the sum takes two: 12 us for 80 tiles in 3 ranges
        const dim3 grid((unsigned)(ntt * ntw * WVT * WVW * (BT / WVT / 16 / QT)));
        if (a.out == kF8BF16) sum_kernel<BT, BW, WVT, WVW, QT, kF8BF16><<<grid, dim3(64), 0, st>>>(a, sp, (int)ntw, vec);
        else sum_kernel<BT, BW, WVT, WVW, QT, kF8F16><<<grid, dim3(64), 0, st>>>(a, sp, (int)ntw, vec);
        HIP_CHECK(hipGetLastError());
    }
}
}  // namespace

bool f8_gemm_takes(const F8Mat& a) {  // rows by index: 32-bit offsets
    return !a.rows || ((int64_t)a.t * a.ldx < (int64_t)1 << 32 && (int64_t)a.t * a.xs_row * 4 < (int64_t)1 << 32);
}
void f8_gemm(const F8Mat& a, int parts, hipStream_t st) {
    if (a.off) gemm_t<256, 256, 2, 4, true>(a, 1, st);
    else gemm_t<256, 256, 2, 4, false>(a, parts, st);
}
