// 8-bit products of few rows (f8.hpp): up to 16 MT rows of one matrix, or of an expert's segment, in one pass over the weights.
// Bound by the weights' bytes. A block holds NT tiles of 16 weight rows; its NW waves share out the 128-k blocks, read their
// weights straight from memory into the matrix core's operands (nothing is shared, so no LDS), and add their sums in the
// order of the waves at the end.
#include "f8.hpp"

namespace {
template <int MT, int NT, int NW, int D, int OUT, bool GROUPED>
__global__ void __launch_bounds__(NW * 64) dec_kernel(F8Mat a, int ntiles, bool vec) {
    __shared__ f32x4_v part[NW * NT * MT * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4, kb = (a.k + 127) >> 7, n16 = (a.n + 15) >> 4;
    const int wt = blockIdx.x % ntiles, job = blockIdx.x / ntiles;
    int e = 0, row0 = job * 16 * MT, rows = min(16 * MT, a.r - row0);
    if constexpr (GROUPED) {
        if (!f8_job<NW * 64>(a.off, a.experts, a.r, 16 * MT, 0, 1, job, reinterpret_cast<int*>(part), e, row0, rows)) return;
        __syncthreads();
    }
    const int n0 = wt * NT;  // first tile of 16 weight rows
    const uint8_t* wp[NT];
#pragma unroll
    for (int i = 0; i < NT; i++)
        wp[i] = static_cast<const uint8_t*>(a.q) + (((size_t)e * n16 + min(n0 + i, n16 - 1)) * kb) * 2048 + lane * 16;
    const float* sw = a.s + ((size_t)e * ((a.n + 127) >> 7) + (n0 >> 3)) * kb;
    const uint8_t* xp[MT];
    const float* sx[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        int64_t row = row0 + min(16 * m + r, rows - 1);
        if (GROUPED && a.rows) {
            row = a.rows[row];
            if ((uint64_t)row >= (uint64_t)a.t) row = 0;  // an index outside x: zeros in y
        }
        xp[m] = static_cast<const uint8_t*>(a.x) + row * a.ldx;
        sx[m] = a.xs + row * a.xs_row;
    }
    // D blocks of 128 k on their way; past the last one the last again, with a scale of zero
    f32x4_v acc[NT][MT] = {};
    i32x8_f8 w[D][NT], x[D][MT];
    float s[D][MT], swb[D];
    auto load = [&](int d, int b) {
        swb[d] = b < kb ? sw[b] : 0.f;
        b = min(b, kb - 1);
        const int at = b * 128 + g * 16, lo = at < a.k ? at : b * 128, hi = at + 64 < a.k ? at + 64 : b * 128;  // behind k the block's first
#pragma unroll
        for (int i = 0; i < NT; i++)
            w[d][i] = f8_join(*reinterpret_cast<const i32x4_f8*>(wp[i] + (size_t)b * 2048), *reinterpret_cast<const i32x4_f8*>(wp[i] + (size_t)b * 2048 + 1024));
#pragma unroll
        for (int m = 0; m < MT; m++) {
            x[d][m] = f8_join(*reinterpret_cast<const i32x4_f8*>(xp[m] + lo), *reinterpret_cast<const i32x4_f8*>(xp[m] + hi));
            s[d][m] = sx[m][b * a.xs_group];
        }
    };
#pragma unroll
    for (int d = 0; d < D - 1; d++) load(d, wave + d * NW);
    for (int b0 = wave; b0 < kb; b0 += D * NW) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            load((d + D - 1) % D, b0 + (d + D - 1) * NW);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const float f = s[d][m] * swb[d];
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const f32x4_v p = f8_mfma(w[d][i], x[d][m]);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][m][j] = fmaf(p[j], f, acc[i][m][j]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int m = 0; m < MT; m++) part[((wave * NT + i) * MT + m) * 64 + lane] = acc[i][m];
    __syncthreads();
    for (int j = tid; j < NT * MT * 64; j += NW * 64) {
        f32x4_v v = part[j];
#pragma unroll
        for (int w = 1; w < NW; w++) {
            const f32x4_v p = part[w * NT * MT * 64 + j];
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] += p[c];
        }
        const int l = j & 63, m = (j >> 6) % MT, i = (j >> 6) / MT, row = 16 * m + (l & 15), col = (n0 + i) * 16 + 4 * (l >> 4);
        if (row >= rows || col >= a.n) continue;
        if (GROUPED && a.rows && (unsigned)a.rows[row0 + row] >= (unsigned)a.t) v = f32x4_v{0.f, 0.f, 0.f, 0.f};
        f8_store4<OUT>(static_cast<uint16_t*>(a.y) + (int64_t)(row0 + row) * a.ldy, col, a.n, v, vec);
    }
}

template <int MT, int NT, int NW, int D, bool GROUPED>
void dec_t(const F8Mat& a, hipStream_t st) {
    const int ntiles = ((a.n + 15) / 16 + NT - 1) / NT;
    const int64_t jobs = GROUPED ? f8_most_jobs(a.r, a.experts, 16 * MT) : (a.r + 16 * MT - 1) / (16 * MT);
    CHECK(jobs * ntiles <= kF8MaxBlocks, "matmul_f8: %lld row blocks by %d column blocks are too many for a call", (long long)jobs, ntiles);
    const dim3 grid((unsigned)(jobs * ntiles)), block(NW * 64);
    const bool vec = f8_vec_ok(a.y, a.ldy);
    if (a.out == kF8BF16) dec_kernel<MT, NT, NW, D, kF8BF16, GROUPED><<<grid, block, 0, st>>>(a, ntiles, vec);
    else dec_kernel<MT, NT, NW, D, kF8F16, GROUPED><<<grid, block, 0, st>>>(a, ntiles, vec);
    HIP_CHECK(hipGetLastError());
}
}  // namespace

// us for 5120 x 17408 with one row: two tiles a block 17.1 (one: 18.3, four: 26.7), loads a step ahead 17.7; 34816 x 5120 with one
// row 31 to 32 by any of these, with 16 rows 35.8 (four waves; eight: 38.9); 160 rows of 512 matrices of 1024 x 2048 43.5 (eight waves; four:
// 44.6, four tiles: 45).
void f8_dec(const F8Mat& a, hipStream_t st) {
    if (a.off) dec_t<1, 2, 8, 1, true>(a, st);
    else if (a.n >= 16384) dec_t<1, 2, 4, 1, false>(a, st);
    else dec_t<1, 2, 8, 1, false>(a, st);
}
