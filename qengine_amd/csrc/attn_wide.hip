// Attention of drafted tokens over the paged cache where a kv head has more rows (drafted tokens times the group's query
// heads) than attn_tree.hip holds beside its keys.
//
// The waves of a block take 32 rows each (attn_wave.hpp) and share 64 keys a step in LDS, so keys and values are read from
// HBM once for 32 W rows. Steps are staged by LDS DMA from the pages, STAGES - 1 of them ahead: one block of 8 waves a CU
// keeps three steps (100 KB at d = 128) on their way, blocks of 4 waves one step each. Work is split over the tokens of all
// sequences evenly (attn_tree.hpp), in units of one step. With the join: 12 trees of up to 32 tokens over up to 6000, 160 rows a
// kv head (206 MB) 77 us; 32 sequences of up to 8000 tokens, 40 rows (718 MB) 155 us, 4.6 TB/s; 2 of 131072 tokens, 40 rows,
// d = 256 (472 MB) 109 us, 4.3 TB/s.
#include "attn_tree.hpp"
#include "attn_wave.hpp"

#include <atomic>

namespace qe_tree {
using qe_tile::dma16_at;

// page numbers are read by scalar loads: a vector load would make the compiler wait for the DMAs in flight
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;

template <int DT, int D, int KEYS, int W, int STAGES>
__global__ __launch_bounds__(64 * W, (D == 256 ? 1 : 2)) void wide_kernel(Args a) {
    using L = Tile<D, KEYS>;
    constexpr int ROWS = 32 * W, N = KEYS / L::RK / W, CHUNK = 16;  // pages are at least 16 tokens
    extern __shared__ char lds[];
    static_assert(STAGES * L::STAGE >= kMaxTreeBatch * (int)sizeof(int), "the units of all sequences fit the stages' place");
    int* ends = reinterpret_cast<int*>(lds);
    __shared__ Kept kept;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const unsigned lds32 = (unsigned)(uintptr_t)lds;

    // A DMA instruction takes RK rows; the wave's n-th starts RK n rows behind its first. The lane's piece of K is the same
    // in all of them, that of V in every second one (d = 256) or all.
    const int r_wave = wave * N * L::RK, r_lane = lane / L::CH;
    constexpr int NV = D == 256 ? 2 : 1;
    const uint32_t k_off = (uint32_t)r_lane * (uint32_t)a.token + ((lane % L::CH) ^ L::kx(r_lane)) * 16;
    uint32_t v_off[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) v_off[i] = (uint32_t)r_lane * (uint32_t)a.token + ((lane % L::CH) ^ L::vx(i * L::RK + r_lane)) * 16;
    Wave32<DT, D, KEYS> w;
    w.places(lane);
    if (W > 4 && wave >= W / 2) __builtin_amdgcn_s_setprio(1);  // one of a SIMD's two waves ahead: its softmax beside the other's products

    int u, u_end, b, base;
    if (!my_units<KEYS, ROWS, 64 * W>(a, ends, kept, u, u_end, b, base)) return;
    while (u < u_end) {
        b = __builtin_amdgcn_readfirstlane(b);
        Seq s = seq_at(a, kept, b);
        s.first = __builtin_amdgcn_readfirstlane(s.first);
        s.n = __builtin_amdgcn_readfirstlane(s.n);
        s.total = __builtin_amdgcn_readfirstlane(s.total);
        s.len = __builtin_amdgcn_readfirstlane(s.len);
        s.slot = __builtin_amdgcn_readfirstlane(s.slot);
        if (s.n <= 0) {
            if (!a.part) return;
            b++;
            continue;
        }
        const int units = unit_count<KEYS>(s.total);
        const int rbs = row_blocks<ROWS>(a, s.n);
        Run run;
        if (!run_of(a, base, u, u_end, units, rbs, run)) return;
        const int rows = s.n * a.group, r = run.rb * ROWS + wave * 32 + col, rc = min(r, rows - 1);
        const int hq = run.h * a.group + rc % a.group, node = rc / a.group;
        const bool busy = run.rb * ROWS + wave * 32 < rows;  // the wave has rows
        uint64_t see = a.mask ? a.mask[s.first + node] : ~0ull >> (63 - node);
        const ScalarInts tab = (ScalarInts)(uintptr_t)(a.table + (int64_t)(s.total > 0 ? s.slot : 0) * a.width);
        const char* kh = a.k + (int64_t)run.h * a.head;
        const char* vh = a.v + (int64_t)run.h * a.head;
        const int pmask = (1 << a.shift) - 1;
        static_assert(N * L::RK <= CHUNK && CHUNK % (N * L::RK) == 0, "a wave's rows of a step are in one page");
        constexpr int NCH = KEYS / CHUNK;  // chunks of a step
        uint32_t ring = 0;                 // which chunks of the last 8 steps have a page, NCH bits each
        auto stage = [&](int j) {
            j = __builtin_amdgcn_readfirstlane(j);
            int pg[NCH];
#pragma unroll
            for (int c = 0; c < NCH; c++) pg[c] = tab[min((j * KEYS + c * CHUNK) >> a.shift, a.width - 1)];
            uint32_t bits = 0;
            int mine = 0;
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                const bool ok = j * KEYS + c * CHUNK < s.total && pg[c] >= 0 && pg[c] < a.pages;
                bits |= ok ? 1u << c : 0u;
                if (c == r_wave / CHUNK) mine = ok ? pg[c] : 0;
            }
            ring = (ring & ~(((1u << NCH) - 1) << (j % 8 * NCH))) | bits << (j % 8 * NCH);
            const unsigned at = lds32 + j % STAGES * L::STAGE;
            const int64_t first = (int64_t)mine * a.page + (int64_t)((j * KEYS + r_wave) & pmask) * a.token;
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(kh + first + i * L::RK * a.token, k_off, at + (wave * N + i) * (1024 + L::PAD));
#pragma unroll
            for (int i = 0; i < N; i++) dma16_at(vh + first + i * L::RK * a.token, v_off[i % NV], at + L::KBYTES + (wave * N + i) * 1024);
        };
        const bool whole = run.t0 == 0 && run.t1 == units;
        const int64_t slot = ((int64_t)blockIdx.x * 2 + (run.t0 > 0 ? 0 : 1)) * ROWS + wave * 32 + col;
        char* out = a.out + (int64_t)(s.first + node) * a.o_row + (int64_t)hq * a.o_head + half * 8;
        float* part = a.part + slot * D + half * 4;

        constexpr int AHEAD = STAGES - 1;  // steps that are under way while one is worked on
        auto first_stages = [&] {
#pragma unroll 1
            for (int j = run.t0; j < min(run.t0 + AHEAD, run.t1); j++) stage(j);
        };
        auto land = [&](int j, int pass) {  // step j is in LDS for every wave, and all are done with the stage that the next step takes
            if (run.t1 - j >= AHEAD) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * N * (AHEAD - 1)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (j + AHEAD < run.t1) stage(j + AHEAD);
            if (pass) {
                keep_tile<DT>(lds + j % STAGES * L::STAGE + L::KBYTES, L::VBYTES, pass, tid, 64 * W);
                __syncthreads();
            }
        };
        auto scores = [&](int j) {
            const uint32_t have = ring >> (j % 8 * NCH) & ((1u << NCH) - 1);
            const int tok0 = j * KEYS + 4 * half;
            return w.scores(lds + j % STAGES * L::STAGE, j * KEYS + KEYS > s.len || have != (1u << NCH) - 1, [&](int x, int e) {
                const int tok = tok0 + 32 * x + 8 * (e / 4) + e % 4, t = tok - s.len;
                // no && or ||: the compiler made branches of them and lost the assignment behind one
                const uint32_t drafted = (uint32_t)(tok < s.total) & (uint32_t)(see >> (t & 63));
                return ((have >> (2 * x + e / 8)) & ((uint32_t)(t < 0) | drafted) & 1) != 0;
            });
        };
        w.load_queries(a.q + (int64_t)(s.first + node) * a.q_row + (int64_t)hq * a.q_head, half);
        for (int pass = 0; pass <= kKinds; pass++) {
            w.clear();
            first_stages();
            w.await_queries();
            asm volatile("" : "+v"(see));
            for (int j = run.t0; j < run.t1; j++) {
                land(j, pass);
                if (busy) w.values(lds + j % STAGES * L::STAGE, scores(j), pass, a.scale2);
            }
            w.settle();
            // (also: every wave is done with the stages)
            const bool again = __syncthreads_or(pass == 0 && busy && r < rows && w.bad());
            if (r < rows && (pass > 0 || !again)) {
                if (pass > 1 && whole) {
                    w.store_kind(out, pass);
                } else if (pass > 1) {
                    w.store_kind(part, pass);
                } else {
                    const float l = sum_over_halves(w.l);
                    if (whole) {
                        w.store(out, l == 0.f ? 0.f : 1.f / l);
                        if (a.lse && half == 0) a.lse[(int64_t)(s.first + node) * a.heads + hq] = l == 0.f ? kNegInf : (w.m + log2f(l)) * kLn2;
                    } else {
#pragma unroll
                        for (int d = 0; d < D / 32; d++)
#pragma unroll
                            for (int e = 0; e < 16; e += 4)
                                *reinterpret_cast<float4*>(part + d * 32 + e * 2) = make_float4(w.o[d][e], w.o[d][e + 1], w.o[d][e + 2], w.o[d][e + 3]);
                        if (half == 0) a.ml[slot] = make_float2(w.m, l);
                    }
                }
            }
            if (pass == 0 && !again) break;
        }
        u += run.t1 - run.t0;
        if (u >= base + units * rbs * a.kv_heads) {
            base += units * rbs * a.kv_heads;
            b++;
        }
    }
}

template <int DT, int D, int KEYS, int W, int STAGES>
void launch_wide(const Args& a, int per_cu, hipStream_t st) {
    constexpr int bytes = STAGES * Tile<D, KEYS>::STAGE;
    static_assert((STAGES & (STAGES - 1)) == 0 && STAGES <= 8, "stages by the step's number");
    const auto kernel = wide_kernel<DT, D, KEYS, W, STAGES>;
    static std::atomic<uint64_t> done{0};  // devices on which the kernel may use so much LDS
    int dev = 0;
    HIP_CHECK(hipGetDevice(&dev));
    if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev < 64) done.fetch_or(1ull << dev);
    }
    launch_split<DT, D, KEYS, 32 * W>(a, kernel, 64 * W, bytes, per_cu, st);
}

// 128 rows a block: two blocks a CU, a step of 64 keys each on its way (three blocks of 32 keys: 32 sequences of 8 drafted
// tokens in groups of 5 115 -> 127 us; one block with three steps on their way 129). More rows: one block of 8 waves.
template <int DT>
void wide(const Args& a, int d, hipStream_t st) {
    const int rows = a.max_new * a.group;
    if (d == 64) rows <= 128 ? launch_wide<DT, 64, 64, 4, 4>(a, 2, st) : launch_wide<DT, 64, 64, 8, 4>(a, 1, st);
    else if (d == 128) rows <= 128 ? launch_wide<DT, 128, 64, 4, 2>(a, 2, st) : launch_wide<DT, 128, 64, 8, 4>(a, 1, st);
    else launch_wide<DT, 256, 32, 4, 4>(a, 1, st);
}
void attend_wide(const Args& a, int d, bool f16, hipStream_t st) { f16 ? wide<kAttnF16>(a, d, st) : wide<kAttnBF16>(a, d, st); }
}  // namespace qe_tree
