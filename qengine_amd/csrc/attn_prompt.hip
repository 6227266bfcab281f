// Causal attention over whole prompts, packed without padding, grouped heads.
//
//   o[i] = sum_{j <= i} p_ij v[j],  p_ij = softmax_j(scale q[i] . k[j])
//
// One pass over the keys with the running maximum and sum of the softmax; a block takes BQ = 32 RW rows of one head, a wave
// 32 of them (attn_wave.hpp). KEYS keys at a time lie in LDS, staged by DMA while the step before is worked on. 16384 rows of
// 16 heads over 2, inputs rotating over three sets, by card: d = 128 1014-1064 us (1035-1085 TFLOP/s; MFMA busy 65 %, beside the
// softmax of three waves a SIMD; 12 bytes a lane are spilled), d = 64 587-613 us, d = 256 2.57-2.60 ms (one wave a SIMD: MFMA,
// LDS reads and softmax add up). Short prompts are bounded by the start of a block (dependent reads of the starts, then queries
// and keys: about 4 us).
#include "attn_wave.hpp"
#include "kv_cache.hpp"
#include "seq_rows.hpp"

#include <algorithm>
#include <atomic>

namespace qe_prompt {
using qe_tile::dma16_at;
constexpr int kMaxSeqs = 4096;     // their block counts are kept in LDS

struct Args {
    const char *q, *k, *v;
    char* out;
    float* lse;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // bytes
    const int32_t* cu;
    int nseq, t, heads, kv_heads;
    float scale2;  // log2(e) times the scale: exponentials are powers of two
};

__device__ __forceinline__ int wave_sum(int x) {  // the same in every lane
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8: sums of rows of 16 in their last lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    return __builtin_amdgcn_readlane(x, 15) + __builtin_amdgcn_readlane(x, 31) + __builtin_amdgcn_readlane(x, 47) + __builtin_amdgcn_readlane(x, 63);
}

// RW waves take 32 rows each; KG groups of RW waves take every KG-th step, each with two stages of its own, and the first
// group adds the others' sums at the end (short prompts: the steps of a block follow each other, so its time is theirs).
template <int DT, int D, int KEYS, int RW, int KG>
__global__ __launch_bounds__(64 * RW * KG, (D == 256 ? 1 : KG == 1 && KEYS == 32 ? 3 : 2)) void prompt_kernel(Args a) {
    using L = Tile<D, KEYS>;
    constexpr int W = RW * KG, BQ = 32 * RW;
    extern __shared__ char lds[];  // two stages of K and V tiles; before them the block counts
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;

    // ---- which rows: blocks of all sequences, those with the most keys first
    const int kvh = blockIdx.x % a.heads % a.kv_heads, grp = blockIdx.x % a.heads / a.kv_heads;
    const int head = kvh * (a.heads / a.kv_heads) + grp;
    int slot = blockIdx.x / a.heads, b = 0, qb = 0;
    auto rows_at = [&](int i) { return rows_of(a.cu[i], a.cu[i + 1], a.t); };
    // the first 64 sequences are in every wave's lanes
    RowRange of_lane{0, 0};
    if (lane < a.nseq) of_lane = rows_at(lane);
    const int lane_first = of_lane.first, lane_len = of_lane.n;
    if (a.nseq == 1) {
        qb = (__builtin_amdgcn_readfirstlane(lane_len) + BQ - 1) / BQ - 1 - slot;
        if (qb < 0) return;
    } else {
        int* more = reinterpret_cast<int*>(lds);  // blocks of the sequences from the 65th on
        const int nb = (lane_len + BQ - 1) / BQ;
        if (a.nseq > 64) {
            for (int i = 64 + tid; i < a.nseq; i += 64 * W) more[i - 64] = (rows_at(i).n + BQ - 1) / BQ;
            __syncthreads();
        }
        BlockPlace place;
        const bool there = place_of(slot, [&](int level) {
            int n = add_blocks(0, nb, level);
            for (int i = lane; i < a.nseq - 64; i += 64) n = add_blocks(n, more[i], level);
            return wave_sum(n);
        }, place);
        if (!there) return;
        qb = place.level;
        int rank = place.rank;
        for (int i0 = 0;; i0 += 64) {
            const bool mine = i0 + lane < a.nseq && (i0 == 0 ? nb : more[i0 - 64 + lane]) > qb;
            const uint64_t has = __ballot(mine);
            const int n = __popcll(has);
            if (rank < n) {
                const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
                b = i0 + __ffsll((unsigned long long)__ballot(mine && before == rank)) - 1;
                break;
            }
            rank -= n;
        }
        if (a.nseq > 64) __syncthreads();
    }
    b = __builtin_amdgcn_readfirstlane(b);
    qb = __builtin_amdgcn_readfirstlane(qb);
    const int c0 = b < 64 ? __builtin_amdgcn_readlane(lane_first, b) : __builtin_amdgcn_readfirstlane(rows_at(b).first);
    const int len = b < 64 ? __builtin_amdgcn_readlane(lane_len, b) : __builtin_amdgcn_readfirstlane(rows_at(b).n);
    const int rw = wave % RW, kg = wave / RW;
    const int q0 = qb * BQ, qw = q0 + rw * 32;    // the block's and the wave's first row
    const int row = qw + col;                     // this lane's query

    const unsigned lds32 = (unsigned)(uintptr_t)lds;
    const char* kb = a.k + (int64_t)c0 * a.k_row + (int64_t)kvh * a.k_head;
    const char* vb = a.v + (int64_t)c0 * a.v_row + (int64_t)kvh * a.v_head;
    // A wave instruction fills 1 KB: RK rows; the wave's n-th starts RK n rows behind its first. Lane i lands at piece i, so
    // it loads the piece that belongs there: of K the same in all instructions, of V in every second one (d = 256) or all.
    constexpr int N = KEYS / L::RK / RW, NV = D == 256 ? 2 : 1;
    const int r_wave = rw * N * L::RK, r_lane = lane / L::CH;
    const uint32_t k_off = (uint32_t)r_lane * (uint32_t)a.k_row + ((lane % L::CH) ^ L::kx(r_lane)) * 16;
    uint32_t v_off[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) v_off[i] = (uint32_t)r_lane * (uint32_t)a.v_row + ((lane % L::CH) ^ L::vx(i * L::RK + r_lane)) * 16;
    auto at_of = [&](int j) { return (kg * 2 + j / KG % 2) * L::STAGE; };  // step j is one of the wave's group
    auto stage = [&](int j) {
        j = __builtin_amdgcn_readfirstlane(j);
        const char* ks = kb + (int64_t)(j * KEYS + r_wave) * a.k_row;
        const char* vs = vb + (int64_t)(j * KEYS + r_wave) * a.v_row;
        const unsigned at = lds32 + at_of(j);
        const int over = (j + 1) * KEYS - len;
        if (over <= 0) {
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(ks + i * L::RK * a.k_row, k_off, at + (rw * N + i) * (1024 + L::PAD));
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(vs + i * L::RK * a.v_row, v_off[i % NV], at + L::KBYTES + (rw * N + i) * 1024);
            return;
        }
        // keys past the end re-read the last one (no row sees them)
        const char* k0 = kb + (int64_t)(j * KEYS) * a.k_row;
        const char* v0 = vb + (int64_t)(j * KEYS) * a.v_row;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = r_wave + i * L::RK + r_lane, key = min(r, KEYS - 1 - over);
            dma16_at(k0, (uint32_t)key * (uint32_t)a.k_row + ((lane % L::CH) ^ L::kx(r)) * 16, at + (rw * N + i) * (1024 + L::PAD));
            dma16_at(v0, (uint32_t)key * (uint32_t)a.v_row + ((lane % L::CH) ^ L::vx(r)) * 16, at + L::KBYTES + (rw * N + i) * 1024);
        }
    };
    const int steps = (min(len, q0 + BQ) + KEYS - 1) / KEYS;
    const int mine = qw < len ? (min(len, qw + 32) + KEYS - 1) / KEYS : 0;  // steps with keys that this wave's rows see
    Wave32<DT, D, KEYS> w;
    w.places(lane);
    w.load_queries(a.q + (int64_t)(c0 + min(row, len - 1)) * a.q_row + (int64_t)head * a.q_head, half);
    char* out = a.out + (int64_t)(c0 + row) * a.o_row + (int64_t)head * a.o_head + half * 8;
    // A value that is not finite in a key that some rows of a step must not see makes those rows' sums NaN (0 times it).
    // Ordinary data has none; where sums of the first pass are not finite the block runs again over the finite values and
    // then over each kind of the others (keep_tile).
    for (int pass = 0; pass <= kKinds; pass++) {
        w.clear();
        if (kg < steps) stage(kg);
        w.await_queries();
        for (int i = 0; i < steps; i += KG) {
            const int j = i + kg;
            // every group's step has landed, and all waves are done with the stages that the next ones take
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (j + KG < steps) stage(j + KG);
            char* tile = lds + at_of(j);
            if (pass) {
                if (j < steps) keep_tile<DT>(tile + L::KBYTES, L::VBYTES, pass, tid % (64 * RW), 64 * RW);
                __syncthreads();
            }
            const int first = j * KEYS + 4 * half - row;  // key - row of the lane's first score
            if (j < mine)
                w.values(tile, w.scores(tile, j * KEYS + KEYS - 1 > qw, [&](int x, int e) { return first + 32 * x + 8 * (e / 4) + e % 4 <= 0; }),
                         pass, a.scale2);
        }
        w.settle();
        if constexpr (KG > 1) w.add_groups(reinterpret_cast<float*>(lds), rw, kg, RW, KG, lane, pass);
        // (also: every wave is done with the stages)
        const bool again = __syncthreads_or(pass == 0 && kg == 0 && row < len && w.bad());
        if (pass > 1) {
            if (kg == 0 && row < len) w.store_kind(out, pass);
        } else if (!again) {
            const float l = sum_over_halves(w.l);
            if (kg == 0 && row < len) {
                w.store(out, l == 0.f ? 0.f : 1.f / l);
                if (a.lse && half == 0) a.lse[(int64_t)(c0 + row) * a.heads + head] = l == 0.f ? kNegInf : (w.m + log2f(l)) * kLn2;
            }
            if (pass == 0) return;
        }
    }
}

template <int DT, int D, int KEYS, int RW, int KG>
void launch(const Args& a, hipStream_t st) {
    constexpr int BQ = 32 * RW, bytes = 2 * KG * Tile<D, KEYS>::STAGE;
    static_assert(bytes >= kMaxSeqs * (int)sizeof(int) && bytes >= Wave32<DT, D, KEYS>::group_bytes(RW, KG), "block counts and groups' sums fit");
    const int64_t blocks = ((int64_t)a.t / BQ + a.nseq) * a.heads;
    CHECK(blocks < (int64_t)1 << 31, "qe_attn_prompt: %lld blocks", (long long)blocks);
    const auto kernel = prompt_kernel<DT, D, KEYS, RW, KG>;
    static std::atomic<uint64_t> done{0};  // devices on which the kernel may use so much LDS
    int dev = 0;
    HIP_CHECK(hipGetDevice(&dev));
    if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev < 64) done.fetch_or(1ull << dev);
    }
    kernel<<<(int)blocks, 64 * RW * KG, bytes, st>>>(a);
    HIP_CHECK(hipGetLastError());
}

template <int DT>
void by_shape(const Args& a, int d, hipStream_t st) {
    // Blocks of 64 rows in four (two for d = 256) groups that share out the keys, while they fill the CUs once, or twice where
    // prompts are long: a block's time is its steps, of which the last rows' has most. us, blocks of 128 rows (steps of 64
    // keys) / these, inputs rotating over three sets: d = 128, 8 heads over 1: 1000 rows 25.4 / 16.6, 2000 44.3 / 26.0, 4000
    // 82 / 54, 40 heads over 8: 300 rows 11.6 / 10.5, 500 16.7 / 18.1, 1000 29.0 / 35.4; d = 256, 16 heads over 2: 1000 48.6 /
    // 38.7, 2000 86 / 78, 4000 181 / 255; d = 64, 8 heads over 1: 2000 31.4 / 16.2 (6000 rows, past the rule, 86 / 68).
    const int64_t blocks = ((int64_t)a.t / 64 + a.nseq) * a.heads, cus = qe_num_cus();
    const bool few = blocks <= cus || (blocks <= 2 * cus && a.t >= (int64_t)1000 * a.nseq);
    // Else blocks of 128 rows. Steps of 32 keys take registers and LDS for three blocks a CU instead of two: us of 64 / 32
    // keys, 40 heads over 8, the same way: d = 128 20 prompts of 8191 rows together, uniformly mixed, 105 / 98, 64 of 128 73 /
    // 64, 4 of 2048 199 / 191, one of 8192 644 / 630; d = 64 the 20 59.5 / 56.4, 4 of 2048 114.9 / 113.2, one of 8192 365 / 373
    // (one of 1000, which the rule gives steps of 32, 19.7 / 23.1).
    const bool lengthy = a.t >= (int64_t)2000 * a.nseq;
    const bool loose = ((int64_t)a.t / 128 + a.nseq) * a.heads <= 2 * cus;  // a block's own time counts: 1000 rows 29.0 / 31.4
    if (d == 64) few ? launch<DT, 64, 64, 2, 4>(a, st) : lengthy ? launch<DT, 64, 64, 4, 1>(a, st) : launch<DT, 64, 32, 4, 1>(a, st);
    else if (d == 128) few ? launch<DT, 128, 32, 2, 4>(a, st) : loose ? launch<DT, 128, 64, 4, 1>(a, st) : launch<DT, 128, 32, 4, 1>(a, st);
    else few ? launch<DT, 256, 32, 2, 2>(a, st) : launch<DT, 256, 64, 4, 1>(a, st);
}
}  // namespace qe_prompt

void attn_prompt(const AttnPromptArgs& x, bool f16, hipStream_t st) {
    CHECK(x.d == 64 || x.d == 128 || x.d == 256, "qe_attn_prompt: d %d (64, 128 or 256)", x.d);
    CHECK(x.kv_heads >= 1 && x.heads >= x.kv_heads && x.heads % x.kv_heads == 0 && x.heads <= 65535, "qe_attn_prompt: %d heads over %d",
          x.heads, x.kv_heads);
    CHECK(x.nseq >= 0 && x.nseq <= qe_prompt::kMaxSeqs && x.t >= 0 && x.t <= kMaxRows, "qe_attn_prompt: nseq %d (at most %d), t %d (at most 2^30)",
          x.nseq, qe_prompt::kMaxSeqs, x.t);
    CHECK(x.scale >= 0x1p-126f && x.scale <= 0x1p126f, "qe_attn_prompt: scale %g", (double)x.scale);
    if (x.nseq == 0 || x.t == 0) return;
    CHECK(x.q && x.k && x.v && x.out && x.cu, "qe_attn_prompt: null pointer");
    CHECK((((uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v | (uintptr_t)x.out) & 15) == 0 &&
              ((x.q_row | x.q_head | x.k_row | x.k_head | x.v_row | x.v_head | x.o_row | x.o_head) & 7) == 0,
          "qe_attn_prompt: q, k, v and out must be 16-byte aligned with strides of 8 elements");
    CHECK(x.k_row >= 0 && x.v_row >= 0 && x.k_row < 1 << 24 && x.v_row < 1 << 24, "qe_attn_prompt: rows of k %lld and v %lld elements apart (below 2^24)",
          (long long)x.k_row, (long long)x.v_row);
    qe_prompt::Args a{(const char*)x.q, (const char*)x.k, (const char*)x.v, (char*)x.out, x.lse,
                      2 * x.q_row, 2 * x.q_head, 2 * x.k_row, 2 * x.k_head, 2 * x.v_row, 2 * x.v_head, 2 * x.o_row, 2 * x.o_head,
                      x.cu, x.nseq, x.t, x.heads, x.kv_heads, x.scale * kLog2e};
    if (f16) qe_prompt::by_shape<kAttnF16>(a, x.d, st);
    else qe_prompt::by_shape<kAttnBF16>(a, x.d, st);
}
