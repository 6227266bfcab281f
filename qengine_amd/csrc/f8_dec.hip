// 8-bit products of few rows (f8.hpp): 16 rows at a time of one matrix, or of an expert's segment, in one pass over the weights.
// Bound by the weights' bytes. A block holds NT tiles of 16 weight rows; its NW waves share out the 128-k blocks, read their
// weights straight from memory into the matrix core's operands (nothing is shared, so no LDS), and add their sums in the
// order of the waves at the end.
#include "f8.hpp"

namespace {
template <int NT, int NW, int OUT, bool GROUPED>
__global__ void __launch_bounds__(NW * 64) dec_kernel(F8Mat a, int ntiles, bool vec) {
    __shared__ f32x4_v part[NW * NT * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4, kb = (a.k + 127) >> 7, n16 = (a.n + 15) >> 4;
    const int wt = blockIdx.x % ntiles, job = blockIdx.x / ntiles;
    int e = 0, row0 = job * 16, rows = min(16, a.r - row0);
    if constexpr (GROUPED) {
        if (!f8_job<NW * 64>(a.off, a.experts, a.r, 16, 0, 1, job, reinterpret_cast<int*>(part), e, row0, rows)) return;
        __syncthreads();
    }
    const int n0 = wt * NT;  // first tile of 16 weight rows
    const uint8_t* wp[NT];
#pragma unroll
    for (int i = 0; i < NT; i++)
        wp[i] = static_cast<const uint8_t*>(a.q) + (((size_t)e * n16 + min(n0 + i, n16 - 1)) * kb) * 2048 + lane * 16;
    const float* sw = a.s + ((size_t)e * ((a.n + 127) >> 7) + (n0 >> 3)) * kb;
    int64_t from = row0 + min(r, rows - 1);
    if (GROUPED && a.rows) {
        from = a.rows[from];
        if ((uint64_t)from >= (uint64_t)a.t) from = 0;  // an index outside x: zeros in y
    }
    const uint8_t* xp = static_cast<const uint8_t*>(a.x) + from * a.ldx;
    const float* sx = a.xs + from * a.xs_row;
    f32x4_v acc[NT] = {};
    for (int b = wave; b < kb; b += NW) {
        const int at = b * 128 + g * 16, lo = at < a.k ? at : b * 128, hi = at + 64 < a.k ? at + 64 : b * 128;  // behind k the block's first
        i32x8_f8 w[NT];
#pragma unroll
        for (int i = 0; i < NT; i++)
            w[i] = f8_join(*reinterpret_cast<const i32x4_f8*>(wp[i] + (size_t)b * 2048), *reinterpret_cast<const i32x4_f8*>(wp[i] + (size_t)b * 2048 + 1024));
        const i32x8_f8 x = f8_join(*reinterpret_cast<const i32x4_f8*>(xp + lo), *reinterpret_cast<const i32x4_f8*>(xp + hi));
        const float f = sx[b * a.xs_group] * sw[b];
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const f32x4_v p = f8_mfma(w[i], x);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = fmaf(p[j], f, acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) part[(wave * NT + i) * 64 + lane] = acc[i];
    __syncthreads();
    for (int j = tid; j < NT * 64; j += NW * 64) {
        f32x4_v v = part[j];
#pragma unroll
        for (int w = 1; w < NW; w++) {
            const f32x4_v p = part[w * NT * 64 + j];
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] += p[c];
        }
        const int l = j & 63, row = l & 15, col = (n0 + (j >> 6)) * 16 + 4 * (l >> 4);
        if (row >= rows || col >= a.n) continue;
        if (GROUPED && a.rows && (unsigned)a.rows[row0 + row] >= (unsigned)a.t) v = f32x4_v{0.f, 0.f, 0.f, 0.f};
        f8_store4<OUT>(static_cast<uint16_t*>(a.y) + (int64_t)(row0 + row) * a.ldy, col, a.n, v, vec);
    }
}

template <int NT, int NW, bool GROUPED>
void dec_t(const F8Mat& a, hipStream_t st) {
    const int ntiles = ((a.n + 15) / 16 + NT - 1) / NT;
    const int64_t jobs = GROUPED ? f8_most_jobs(a.r, a.experts, 16) : (a.r + 15) / 16;
    CHECK(jobs * ntiles <= kF8MaxBlocks, "matmul_f8: %lld row blocks by %d column blocks are too many for a call", (long long)jobs, ntiles);
    const dim3 grid((unsigned)(jobs * ntiles)), block(NW * 64);
    const bool vec = f8_vec_ok(a.y, a.ldy);
    if (a.out == kF8BF16) dec_kernel<NT, NW, kF8BF16, GROUPED><<<grid, block, 0, st>>>(a, ntiles, vec);
    else dec_kernel<NT, NW, kF8F16, GROUPED><<<grid, block, 0, st>>>(a, ntiles, vec);
    HIP_CHECK(hipGetLastError());
}
}  // namespace

// us by two tiles and eight waves a block / one tile / four tiles / two tiles and four waves, weights rotating over three sets: one row of
// 5120 x 17408 15.9 / 16.5 / 24.4 / 23.8, 16 rows 19.0 / 27.0 / 28.6 / 25.0; one row of 34816 x 5120 32.5 / 31.0 / 35.0 / 32.9, 16 rows 36.1 / 41.8 /
// 38.2 / 36.0; 160 rows of 512 matrices of 1024 x 2048 47.8 / 61.6 / 48.9 / 48.3.
void f8_dec(const F8Mat& a, hipStream_t st) {
    if (a.off) dec_t<2, 8, true>(a, st);
    else if (a.n >= 16384) dec_t<2, 4, false>(a, st);
    else dec_t<2, 8, false>(a, st);
}
