// Causal attention over whole prompts, packed without padding, grouped heads.
//
//   o[i] = sum_{j <= i} p_ij v[j],  p_ij = softmax_j(scale q[i] . k[j])
//
// One pass over the keys with the running maximum and sum of the softmax; a block takes BQ = 32 W rows of one head, a wave
// 32 of them with its queries, its scores S^T = K Q^T (32 x 32 x 16 MFMA) and its sums O^T = V^T P^T in registers. 64 keys
// at a time lie in LDS, staged by LDS DMA while the 64 before are worked on. A wave reads K as the A operand in 16-byte
// pieces and V's transpose by ds_read_b64_tr_b16; both tiles are stored with their 16-byte pieces permuted by row so that
// these reads meet no bank twice.
#include "attn_common.hpp"
#include "kv_cache.hpp"
#include "mfma_tile.hpp"

#include <algorithm>
#include <atomic>

namespace qe_prompt {
using qe_tile::dma16_at;
constexpr int kKeys = 64;          // keys of a step
constexpr int kMaxSeqs = 4096;     // their block counts are kept in LDS
constexpr float kLazy = 8.f;       // the running maximum follows a row's scores once they pass it by this much (2^8 in the sums)

struct Args {
    const char *q, *k, *v;
    char* out;
    float* lse;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // bytes
    const int32_t* cu;
    int nseq, t, heads, kv_heads;
    float scale2;  // log2(e) times the scale: exponentials are powers of two
};

// Tiles in LDS. A row is CH = D / 8 pieces of 16 bytes, a DMA instruction fills 1 KB = RK rows.
// K: a wave reads one piece of 32 rows (ds_read_b128), so 16 neighbouring rows must have it in 16 different places of a
// 256-byte line: pieces are permuted inside groups of 1, 2 or 4 by row, and each KB starts PAD bytes further on.
// V: a transposing read (ds_read_b64_tr_b16) takes 64 bytes of 8 rows, 4 rows at a time: the 64-byte windows of a row are
// permuted by row.
// Both permutations touch few bits, so a lane's addresses are one to four bases and constants.
template <int D>
struct Tile {
    static constexpr int KEYS = kKeys, CH = D / 8, RK = 64 / CH, PAD = D == 256 ? 32 : 64;
    static constexpr int KBYTES = KEYS / RK * (1024 + PAD), VBYTES = KEYS * D * 2, STAGE = KBYTES + VBYTES;
    static __device__ __forceinline__ int kx(int r) { return D == 256 ? r & 1 : D == 128 ? r & 3 : r >> 1 & 3; }
    static __device__ __forceinline__ int vx(int r) { return (D == 64 ? r >> 1 & 1 : r & 3) << 2; }
    static __device__ __forceinline__ int k_row(int r) { return r / RK * (1024 + PAD) + r % RK * (D * 2); }
};

__device__ __forceinline__ int wave_sum(int x) {  // the same in every lane
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8: sums of rows of 16 in their last lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    return __builtin_amdgcn_readlane(x, 15) + __builtin_amdgcn_readlane(x, 31) + __builtin_amdgcn_readlane(x, 47) + __builtin_amdgcn_readlane(x, 63);
}

template <int DT, int D, int W>
__global__ __launch_bounds__(64 * W, (D == 256 ? 1 : 2)) void prompt_kernel(Args a) {
    using T = AttnT<DT>;
    constexpr int BQ = 32 * W, KS = D / 16, DB = D / 32, KEYS = kKeys, NX = KEYS / 32;
    using L = Tile<D>;
    extern __shared__ char lds[];  // two stages of K and V tiles; before them the block counts
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;

    // ---- which rows: blocks of all sequences, those with the most keys first
    const int kvh = blockIdx.x % a.heads % a.kv_heads, grp = blockIdx.x % a.heads / a.kv_heads;
    const int head = kvh * (a.heads / a.kv_heads) + grp;
    int slot = blockIdx.x / a.heads, b = 0, qb = 0;
    auto blocks_of = [&](int i) {
        const int c0 = min(max(a.cu[i], 0), a.t), c1 = min(a.cu[i + 1], a.t);
        return c1 > c0 ? (c1 - c0 + BQ - 1) / BQ : 0;
    };
    if (a.nseq == 1) {
        qb = blocks_of(0) - 1 - slot;
        if (qb < 0) return;
    } else {
        int* more = reinterpret_cast<int*>(lds);  // blocks of the sequences from the 65th on; every wave holds the first 64
        const int nb = lane < a.nseq ? blocks_of(lane) : 0;
        if (a.nseq > 64) {
            for (int i = 64 + tid; i < a.nseq; i += 64 * W) more[i - 64] = blocks_of(i);
            __syncthreads();
        }
        // blocks with index >= level, over all sequences
        auto count = [&](int level) {
            int n = max(0, nb - level);
            for (int i = lane; i < a.nseq - 64; i += 64) n += max(0, more[i] - level);
            return wave_sum(n);
        };
        int lo = 0, above = 0;  // the largest level with more than `slot` blocks from it on, and the blocks above it
        int hi = 1;
        if (slot >= count(0)) return;
        for (int n; (n = count(hi)) > slot; hi *= 2) lo = hi;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (count(mid) > slot) lo = mid;
            else hi = mid;
        }
        above = count(lo + 1);
        qb = lo;
        int rank = slot - above;  // among the sequences that have a block of this index
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
    const int c0 = min(max(a.cu[b], 0), a.t), len = min(a.cu[b + 1], a.t) - c0;
    const int q0 = qb * BQ, qw = q0 + wave * 32;  // the block's and the wave's first row
    const int row = qw + col;                     // this lane's query

    const unsigned lds32 = (unsigned)(uintptr_t)lds;
    const char* kb = a.k + (int64_t)c0 * a.k_row + (int64_t)kvh * a.k_head;
    const char* vb = a.v + (int64_t)c0 * a.v_row + (int64_t)kvh * a.v_head;
    // a wave instruction fills 1 KB: RK rows; lane i lands at piece i, so it loads the piece that belongs there
    constexpr int N = KEYS / L::RK / W;
    uint32_t k_off[N], v_off[N];  // of a step's first key
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int r = (wave * N + i) * L::RK + lane / L::CH;
        k_off[i] = (uint32_t)r * (uint32_t)a.k_row + ((lane % L::CH) ^ L::kx(r)) * 16;
        v_off[i] = (uint32_t)r * (uint32_t)a.v_row + ((lane % L::CH) ^ L::vx(r)) * 16;
    }
    auto stage = [&](int j, int buf) {
        const char* ks = kb + (int64_t)j * KEYS * a.k_row;
        const char* vs = vb + (int64_t)j * KEYS * a.v_row;
        const unsigned at = lds32 + buf * L::STAGE;
        const int over = (j + 1) * KEYS - len;
        if (over <= 0) {
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(ks, k_off[i], at + (wave * N + i) * (1024 + L::PAD));
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(vs, v_off[i], at + L::KBYTES + (wave * N + i) * 1024);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {  // keys past the end re-read the last one (no row sees them)
            const uint32_t back = max(0, (wave * N + i) * L::RK + lane / L::CH + over - (KEYS - 1));
            dma16_at(ks, k_off[i] - back * (uint32_t)a.k_row, at + (wave * N + i) * (1024 + L::PAD));
            dma16_at(vs, v_off[i] - back * (uint32_t)a.v_row, at + L::KBYTES + (wave * N + i) * 1024);
        }
    };
    const int steps = (min(len, q0 + BQ) + KEYS - 1) / KEYS;
    const int mine = qw < len ? (min(len, qw + 32) + KEYS - 1) / KEYS : 0;  // steps with keys that this wave's rows see
    stage(0, 0);
    // The queries are waited for here: a use inside the loop would make the compiler wait there for whatever loads are in
    // flight, which are the next step's.
    u32x4_v q[KS];
    {
        const char* p = a.q + (int64_t)(c0 + min(row, len - 1)) * a.q_row + (int64_t)head * a.q_head + half * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] = *reinterpret_cast<const u32x4_v*>(p + ks * 32);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(q[ks]));
    }
    // a lane's places in a K tile (row col, piece 2 ks + half for ks = 0 and 1) and in a V tile (row 4 half + (0 .. 3) by lane,
    // columns 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) for d = 0 .. 3)
    int kat[2], vat[4];
#pragma unroll
    for (int i = 0; i < 2; i++) kat[i] = L::k_row(col) + (((2 * i + half) ^ L::kx(col)) * 16);
    {
        const int vr = 4 * half + (lane & 15) / 4, vc = (lane >> 4 & 1) * 2 + (lane & 3) / 2;
#pragma unroll
        for (int d = 0; d < 4; d++) vat[d] = L::KBYTES + vr * D * 2 + (((4 * d + vc) ^ L::vx(vr)) * 16) + (lane & 1) * 8;
    }
    f32x16_v o[DB];
    float m, l;
    // A value that is not finite in a key that some rows of a step must not see makes those rows' sums NaN (0 times it).
    // Ordinary data has none; where sums of the first pass are not finite the block runs again, value by value of kKinds:
    // over the finite values alone, then over ones in the place of each kind of the others, weighted 1 where a row sees the
    // key, which tells the outputs that are +inf, -inf or NaN.
    for (int pass = 0;; pass++) {
        m = kNegInf;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.f;
        if (pass) stage(0, 0);
        for (int j = 0; j < steps; j++) {
            // step j has landed everywhere, and every wave is done with the stage that step j + 1 goes to
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (j + 1 < steps) stage(j + 1, (j + 1) & 1);
            char* tile = lds + (j & 1) * L::STAGE;
            if (pass) {
                keep_tile<DT>(tile + L::KBYTES, L::VBYTES, pass, tid, 64 * W);
                __syncthreads();
            }
            if (j >= mine) continue;
            // operands are read in groups, a group ahead of the products that use it; the sums of one V group follow the
            // last scores' products, so that its reads are under way during the softmax
            constexpr int GK = 8, NK = NX * KS / GK, GV = 4, NV = DB * 2 * NX / GV;
            u32x4_v kf[2][GK], vf[2][GV];
            auto read_k = [&](int g) {
#pragma unroll
                for (int i = 0; i < GK; i++) {
                    const int x = (g * GK + i) % NX, ks = (g * GK + i) / NX;
                    constexpr int M = D == 256 ? 1 : 2;  // bases
                    const int at = kat[ks % M] + ks / M * M * 32 + 32 / L::RK * (1024 + L::PAD) * x;
                    kf[g % 2][i] = *reinterpret_cast<const u32x4_v*>(tile + at);
                }
            };
            auto read_v = [&](int g) {
#pragma unroll
                for (int i = 0; i < GV; i++) {
                    const int d = (g * GV + i) / (2 * NX), y = (g * GV + i) % (2 * NX);
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        const int at = vat[d % 4] + d / 4 * 256 + (16 * y + 8 * z) * D * 2;
                        const s16x4_v w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_v*)(tile + at));
                        const uint2 w2 = __builtin_bit_cast(uint2, w);
                        vf[g % 2][i][2 * z] = w2.x;
                        vf[g % 2][i][2 * z + 1] = w2.y;
                    }
                }
            };
            f32x16_v s[NX];
#pragma unroll
            for (int x = 0; x < NX; x++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[x][e] = 0.f;
            read_k(0);
#pragma unroll
            for (int g = 0; g < NK; g++) {
                if (g + 1 < NK) read_k(g + 1);
                else read_v(0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < GK; i++) s[(g * GK + i) % NX] = T::mfma32(kf[g % 2][i], q[(g * GK + i) / NX], s[(g * GK + i) % NX]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // a lane's scores: keys j KEYS + 32 x + 8 (e / 4) + 4 half + e % 4 of its query
            if (j * KEYS + KEYS - 1 > qw) {
                const int first = j * KEYS + 4 * half - row;  // key - row of the lane's first score
#pragma unroll
                for (int x = 0; x < NX; x++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (first + 32 * x + 8 * (e / 4) + e % 4 > 0) s[x][e] = kNegInf;
            }
            float mx = kNegInf;
#pragma unroll
            for (int x = 0; x < NX; x++)
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[x][e]);
            mx *= a.scale2;
            if (__any(mx > m + kLazy)) {
                const float top = fmaxf(m, max_over_halves(mx));
                const float f0 = top == kNegInf || pass > 1 ? 1.f : __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= f0;
#pragma unroll
                for (int d = 0; d < DB; d++) o[d] *= f0;
            }
            const float base = m == kNegInf ? 0.f : m;
            u32x4_v p[2 * NX];
#pragma unroll
            for (int x = 0; x < NX; x++)
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], a.scale2, -base));
                    const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e + 1], a.scale2, -base));
                    l += w0 + w1;
                    p[2 * x + e / 8][e % 8 / 2] = T::pack(w0, w1);
                }
            if (pass > 1) {
#pragma unroll
                for (int x = 0; x < NX; x++)
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        p[2 * x + e / 8][e % 8 / 2] = (s[x][e] != kNegInf ? T::kOne : 0u) | (s[x][e + 1] != kNegInf ? T::kOne << 16 : 0u);
            }
            // V^T's operand: 32 columns, 16 keys in the order of the scores: 4 half + (0 .. 3) and 8 more
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < NV; g++) {
                if (g + 1 < NV) read_v(g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < GV; i++) {
                    const int d = (g * GV + i) / (2 * NX);
                    o[d] = T::mfma32(vf[g % 2][i], p[(g * GV + i) % (2 * NX)], o[d]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        bool again = false;
        if (pass == 0) {
            float bad = 0.f;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) bad = __builtin_fmaf(o[d][e], 0.f, bad);
            again = row < len && !(bad == 0.f);
        }
        // (also: every wave is done with the stages)
        again = __syncthreads_or(again) || pass > 0;
        char* p = a.out + (int64_t)(c0 + row) * a.o_row + (int64_t)head * a.o_head + half * 8;
        if (pass > 1) {
            if (row < len)
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        uint16_t* at = reinterpret_cast<uint16_t*>(p + d * 64 + e / 4 * 16 + e % 4 * 2);
                        if (o[d][e] > 0.f) *at = add_kind<DT>(*at, pass);
                    }
            if (pass == kKinds) return;
            continue;
        }
        if (pass == 0 && again) continue;
        l = sum_over_halves(l);
        if (row < len) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    uint2 w;
                    w.x = T::pack(o[d][e] * inv, o[d][e + 1] * inv);
                    w.y = T::pack(o[d][e + 2] * inv, o[d][e + 3] * inv);
                    *reinterpret_cast<uint2*>(p + d * 64 + e * 4) = w;
                }
            if (a.lse && half == 0) a.lse[(int64_t)(c0 + row) * a.heads + head] = l == 0.f ? kNegInf : (m + log2f(l)) * kLn2;
        }
        if (!again) return;
    }
}

template <int DT, int D, int W>
void launch(const Args& a, hipStream_t st) {
    constexpr int BQ = 32 * W;
    const int64_t blocks = ((int64_t)a.t / BQ + a.nseq) * a.heads;
    CHECK(blocks < (int64_t)1 << 31, "qe_attn_prompt: %lld blocks", (long long)blocks);
    const int bytes = std::max(2 * Tile<D>::STAGE, a.nseq * 4);
    if (bytes > 64 * 1024) {
        static std::atomic<uint64_t> done{0};  // per device, one bit
        int dev = 0;
        HIP_CHECK(hipGetDevice(&dev));
        if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
            HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(prompt_kernel<DT, D, W>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            if (dev < 64) done.fetch_or(1ull << dev);
        }
    }
    prompt_kernel<DT, D, W><<<(int)blocks, 64 * W, bytes, st>>>(a);
    HIP_CHECK(hipGetLastError());
}

template <int DT>
void by_shape(const Args& a, int d, hipStream_t st) {
    if (d == 64) launch<DT, 64, 4>(a, st);
    else if (d == 128) launch<DT, 128, 4>(a, st);
    else launch<DT, 256, 4>(a, st);
}
}  // namespace qe_prompt

void attn_prompt(const AttnPromptArgs& x, bool f16, hipStream_t st) {
    CHECK(x.d == 64 || x.d == 128 || x.d == 256, "qe_attn_prompt: d %d (64, 128 or 256)", x.d);
    CHECK(x.kv_heads >= 1 && x.heads >= x.kv_heads && x.heads % x.kv_heads == 0 && x.heads <= 65535, "qe_attn_prompt: %d heads over %d",
          x.heads, x.kv_heads);
    CHECK(x.nseq >= 0 && x.nseq <= qe_prompt::kMaxSeqs && x.t >= 0, "qe_attn_prompt: nseq %d (at most %d), t %d", x.nseq, qe_prompt::kMaxSeqs, x.t);
    CHECK(x.scale > 0.f && x.scale < __builtin_huge_valf(), "qe_attn_prompt: scale %g", (double)x.scale);
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
