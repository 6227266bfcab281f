// Attention of drafted tokens (one, a chain or a tree) over the paged cache.
//
//   o[i] = sum_j p_ij v[j],  p_ij = softmax over the tokens j that row i sees of scale q[i] . k[j]
//
// A sequence's rows of one kv head are its drafted tokens times the query heads of the group: here few (1 to 32) against
// thousands of keys, so the call is bound by reading keys and values once from HBM. Every wave takes 32 keys at a
// time straight into registers (no LDS: nobody else needs them): K as the A operand of S^T = K Q^T as it lies in memory,
// V's rows 16 bytes a lane, turned into the A operand of O^T = V^T P^T by 16-bit permutes inside the lane (8 keys x 8
// columns: 32 permutes for 32 keys x 128 columns, hidden behind the loads). The next 32 keys are in flight meanwhile:
// 128 KB a CU at d = 128. 64 sequences of up to 8000 tokens, 8 kv heads (1.24 GB): 227 us, 5.5 TB/s.
//
// Work is split over the tokens of all sequences evenly (attn_tree.hpp), in units of 128 tokens, 32 a wave.
#include "attn_tree.hpp"

namespace qe_tree {
constexpr int kWaves = 4, kUnit = 128;

// blocks of the kernel on a CU, by its registers
constexpr int blocks_of(int nt_d) { return nt_d == 64 ? 3 : nt_d == 128 ? 2 : 1; }

template <int D>
struct Frag {  // 32 keys of a wave
    static constexpr int KS = D / 32, VD = D / 32;  // 16-byte pieces of a key row per lane; dwords of a value row per lane
    u32x4_v k[2][KS];
    uint32_t v[8][VD];
    bool ok[2];  // the half's page exists
};

template <int DT, int D, int NT>
__global__ __launch_bounds__(kThreads, blocks_of(NT * D)) void tree_kernel(Args a) {
    using T = AttnT<DT>;
    using F = Frag<D>;
    static_assert(NT * D <= 256, "registers for the next keys and values beside these");
    constexpr int ROWS = 16 * NT, KS = F::KS, VD = F::VD, DT16 = D / 16;
    constexpr int PITCH = D + 4;
    __shared__ float obuf[kWaves][16][PITCH];
    __shared__ float2 mlbuf[kWaves][16];
    static_assert(sizeof(obuf) >= kMaxTreeBatch * sizeof(int), "the units of all sequences fit the sums' place");
    int* ends = reinterpret_cast<int*>(obuf);
    __shared__ Kept kept;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;

    int u, u_end, b, base;
    if (!my_units<kUnit, ROWS, kThreads>(a, ends, kept, u, u_end, b, base)) return;
    while (u < u_end) {
        b = __builtin_amdgcn_readfirstlane(b);
        const Seq s = seq_at(a, kept, b);
        if (s.n <= 0) {
            if (!a.part) return;
            b++;
            continue;
        }
        const int units = unit_count<kUnit>(s.total);
        const int rbs = row_blocks<ROWS>(a, s.n);
        Run run;
        if (!run_of(a, base, u, u_end, units, rbs, run)) return;
        const int h = run.h, rb = run.rb, t0 = run.t0, t1 = run.t1;
        const int rows = s.n * a.group;  // row r: drafted token r / group, query head r % group of the kv head

        // the rows' queries (B operand) and masks
        u32x4_v q[NT][KS];
        uint64_t see[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = rb * ROWS + nt * 16 + col;
            const int rc = min(r, rows - 1), i = rc / a.group, g = rc % a.group;
            const char* p = a.q + (int64_t)(s.first + i) * a.q_row + (int64_t)(h * a.group + g) * a.q_head + grp * 16;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) q[nt][ks] = *reinterpret_cast<const u32x4_v*>(p + ks * 64);
            see[nt] = a.mask ? a.mask[s.first + i] : ~0ull >> (63 - i);
        }
        f32x4_v o[NT][DT16];
        float m[NT], l[NT];
        int pass = 0;

        const int32_t* tab = a.table + (int64_t)s.slot * a.width;
        const char* kh = a.k + (int64_t)h * a.head + col * a.token + grp * 16;
        const char* vh = a.v + (int64_t)h * a.head + 4 * grp * a.token + col * (D == 64 ? 8 : 16);
        const int pmask = (1 << a.shift) - 1;
        auto page_at = [&](int tok) {  // -1: none
            const int i = tok >> a.shift;
            int pg = -1;
            if (tok < s.total) pg = __builtin_amdgcn_readfirstlane(tab[i]);
            return pg >= 0 && pg < a.pages ? pg : -1;
        };
        auto load = [&](F& f, int tb) {  // the 32 tokens from tb (a multiple of 32); pages are at least 16 tokens
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int tok = tb + 16 * x, pg = page_at(tok);
                f.ok[x] = pg >= 0;
                const int64_t off = (int64_t)max(pg, 0) * a.page + (int64_t)(tok & pmask) * a.token;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) f.k[x][ks] = *reinterpret_cast<const u32x4_v*>(kh + off + ks * 64);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const char* p = vh + off + j * a.token;
                    if constexpr (D == 64) {
                        const uint2 w = *reinterpret_cast<const uint2*>(p);
                        f.v[4 * x + j][0] = w.x;
                        f.v[4 * x + j][1] = w.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < VD / 4; c++) {
                            const u32x4_v w = *reinterpret_cast<const u32x4_v*>(p + c * 256);
#pragma unroll
                            for (int e = 0; e < 4; e++) f.v[4 * x + j][4 * c + e] = w[e];
                        }
                    }
                }
            }
        };
        // column block t of V^T: lane's column (its 16-byte piece of the rows, value t), 8 keys
        auto vt = [&](const F& f, int t) {
            u32x4_v r;
#pragma unroll
            for (int p = 0; p < 4; p++)
                r[p] = __builtin_amdgcn_perm(f.v[2 * p + 1][t / 2], f.v[2 * p][t / 2], t % 2 ? 0x07060302u : 0x05040100u);
            return r;
        };
        auto compute = [&](F& f, int tb) {
            f32x4_v sc[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    sc[nt][x] = f32x4_v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) sc[nt][x] = T::mfma16(f.k[x][ks], q[nt][ks], sc[nt][x]);
                }
            const bool masked = tb + 32 > s.len || !f.ok[0] || !f.ok[1];
            if (masked) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int tok = tb + 16 * x + 4 * grp + e, j = tok - s.len;
                            const uint32_t drafted = (uint32_t)(tok < s.total) & (uint32_t)(see[nt] >> (j & 63));
                            const bool on = ((uint32_t)f.ok[x] & ((uint32_t)(j < 0) | drafted) & 1) != 0;
                            sc[nt][x][e] = on ? mul_rounded(sc[nt][x][e], a.scale2) : kNegInf;
                        }
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[nt][x][e] = mul_rounded(sc[nt][x][e], a.scale2);
            }
            u32x4_v p[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float mx = kNegInf;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx = fmaxf(mx, sc[nt][x][e]);
                if (pass == 1) mx += T::kRoom;
                if (__any(mx - m[nt] > kLazy)) {  // (m + kLazy would round up to the next number where that is 2 kLazy away)
                    const float top = fmaxf(m[nt], max_over_quarters(mx));
                    const float f0 = top == kNegInf || pass > 1 ? 1.f : __builtin_amdgcn_exp2f(m[nt] - top);
                    m[nt] = top;
                    l[nt] *= f0;
#pragma unroll
                    for (int t = 0; t < DT16; t++) o[nt][t] *= f0;
                }
                const float base = m[nt] == kNegInf ? 0.f : m[nt];
                float w[8];
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[4 * x + e] = __builtin_amdgcn_exp2f(sc[nt][x][e] - base);
                        l[nt] += w[4 * x + e];
                    }
#pragma unroll
                for (int e = 0; e < 4; e++) p[nt][e] = T::pack(w[2 * e], w[2 * e + 1]);
            }
            if (pass) {
#pragma unroll
                for (int r = 0; r < 8; r++)
#pragma unroll
                    for (int e = 0; e < VD; e++) f.v[r][e] = keep_two<DT>(f.v[r][e], pass);
                if (pass > 1)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            p[nt][e] = (sc[nt][e / 2][e % 2 * 2] != kNegInf ? T::kOne : 0u) |
                                       (sc[nt][e / 2][e % 2 * 2 + 1] != kNegInf ? T::kOne << 16 : 0u);
            }
#pragma unroll
            for (int t = 0; t < DT16; t++) {
                const u32x4_v v = vt(f, t);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) o[nt][t] = T::mfma16(v, p[nt], o[nt][t]);
            }
        };

        // this wave's tokens: 32 of each unit; the next 32 are on their way meanwhile
        const int stop = min(t1 * kUnit, s.total);
        uint32_t kinds[3][NT][(DT16 * 4 + 31) / 32];  // bit: the wave's row sees a +inf, -inf, NaN in the column
        for (;;) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                m[nt] = kNegInf;
                l[nt] = 0.f;
#pragma unroll
                for (int t = 0; t < DT16; t++) o[nt][t] = f32x4_v{0.f, 0.f, 0.f, 0.f};
            }
            int tb = t0 * kUnit + wave * 32;
            if (tb < stop) {
                F f;
                load(f, tb);
                for (; tb < stop; tb += kUnit) {
                    F next;
                    load(next, tb + kUnit < stop ? tb + kUnit : tb);
                    compute(f, tb);
                    f = next;
                }
            }
            if (pass == 0) {
                float bad = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int t = 0; t < DT16; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) bad = if_bad(o[nt][t][e], bad);
                if (!__any(!(bad == 0.f))) break;
                pass = 2;
            } else if (pass > 1) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int w = 0; w < (DT16 * 4 + 31) / 32; w++) {
                        uint32_t bits = 0;
#pragma unroll
                        for (int i = 32 * w; i < 32 * w + 32 && i < DT16 * 4; i++) bits |= o[nt][i / 4][i % 4] > 0.f ? 1u << (i % 32) : 0u;
                        if (pass == 2) kinds[0][nt][w] = bits;
                        else if (pass == 3) kinds[1][nt][w] = bits;
                        else kinds[2][nt][w] = bits;
                    }
                pass = pass == kKinds ? 1 : pass + 1;
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < DT16 * 4; i++) {
                        float y = o[nt][i / 4][i % 4];
                        const uint32_t bit = 1u << (i % 32);
                        if (kinds[0][nt][i / 32] & bit) y += __builtin_huge_valf();
                        if (kinds[1][nt][i / 32] & bit) y -= __builtin_huge_valf();
                        o[nt][i / 4][i % 4] = kinds[2][nt][i / 32] & bit ? __builtin_nanf("") : y;
                    }
                break;
            }
        }

        // join the four waves, 16 rows at a time
        const bool whole = t0 == 0 && t1 == units;
        const int64_t pslot = ((int64_t)blockIdx.x * 2 + (t0 > 0 ? 0 : 1)) * ROWS;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            l[nt] = sum_over_quarters(l[nt]);
            __syncthreads();
            if (lane < 16) mlbuf[wave][col] = make_float2(m[nt], l[nt]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // lane's columns: piece 4 grp + e of 8 (4 for D = 64) columns, 128 further on for the next pieces
#pragma unroll
                for (int t = 0; t < DT16; t += 4) {
                    const int d = D == 64 ? 4 * (4 * grp + e) : 8 * (4 * grp + e) + t % 8 + t / 8 * 128;
                    float4 w = make_float4(o[nt][t][e], o[nt][t + 1][e], o[nt][t + 2][e], o[nt][t + 3][e]);
                    *reinterpret_cast<float4*>(&obuf[wave][col][d]) = w;
                }
            }
            __syncthreads();
            const int row = tid >> 4, c0 = (tid & 15) * (D / 16), r = rb * ROWS + nt * 16 + row;
            float top = kNegInf, sum = 0.f, f[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; w++) top = fmaxf(top, mlbuf[w][row].x);
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float2 x = mlbuf[w][row];
                f[w] = x.x == kNegInf ? 0.f : __builtin_amdgcn_exp2f(x.x - top);
                if (x.x == __builtin_huge_valf()) f[w] = 1.f;  // the row's sums are NaN already
                sum += f[w] * x.y;
                if (x.x != kNegInf) f[w] = above_zero(f[w]);
            }
            float y[D / 16];
#pragma unroll
            for (int d = 0; d < D / 16; d += 4) {
                float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float4 x = *reinterpret_cast<const float4*>(&obuf[w][row][c0 + d]);
                    z.x += f[w] * x.x;
                    z.y += f[w] * x.y;
                    z.z += f[w] * x.z;
                    z.w += f[w] * x.w;
                }
                y[d] = z.x;
                y[d + 1] = z.y;
                y[d + 2] = z.z;
                y[d + 3] = z.w;
            }
            if (r >= rows) continue;
            if (whole) {
                const int i = r / a.group, hq = h * a.group + r % a.group;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                char* p = a.out + (int64_t)(s.first + i) * a.o_row + (int64_t)hq * a.o_head + c0 * 2;
#pragma unroll
                for (int d = 0; d < D / 16; d += 4) {
                    uint2 w;
                    w.x = T::pack(y[d] * inv, y[d + 1] * inv);
                    w.y = T::pack(y[d + 2] * inv, y[d + 3] * inv);
                    *reinterpret_cast<uint2*>(p + d * 2) = w;
                }
                if (a.lse && (tid & 15) == 0) a.lse[(int64_t)(s.first + i) * a.heads + hq] = sum == 0.f ? kNegInf : (top + log2f(sum)) * kLn2;
            } else {
                float* p = a.part + (pslot + nt * 16 + row) * D + c0;
#pragma unroll
                for (int d = 0; d < D / 16; d += 4) *reinterpret_cast<float4*>(p + d) = make_float4(y[d], y[d + 1], y[d + 2], y[d + 3]);
                if ((tid & 15) == 0) a.ml[pslot + nt * 16 + row] = make_float2(top, sum);
            }
        }
        u += t1 - t0;
        if (u >= base + units * rbs * a.kv_heads) {
            base += units * rbs * a.kv_heads;
            b++;
        }
    }
}

template <int DT, int D, int NT>
void launch(const Args& a, hipStream_t st) {
    launch_split<DT, D, kUnit, 16 * NT>(a, tree_kernel<DT, D, NT>, kThreads, 0, blocks_of(NT * D), st);
}

// Few rows of a kv head: this kernel, more: attn_wide.hip. us here / there, 16 sequences of 4600 tokens over 8 kv heads, inputs
// rotating over three sets: d = 64 16 rows a head 39.0 / 44.8, 32 rows 43.8 / 45.6; d = 128 16 rows 67.5 / 63.6, 32 rows 72 / 66.
// 5 rows, d = 128: one sequence of 2100 tokens 11.9 / 12.7, 64 of up to 8000 227 / 224.
template <int DT>
void by_shape(const Args& a, int d, hipStream_t st) {
    const int rows = a.max_new * a.group;
    if (rows > (d == 64 ? 32 : 16)) attend_wide(a, d, DT == kAttnF16, st);
    else if (d == 64) rows <= 16 ? launch<DT, 64, 1>(a, st) : launch<DT, 64, 2>(a, st);
    else if (d == 128) launch<DT, 128, 1>(a, st);
    else launch<DT, 256, 1>(a, st);
}
}  // namespace qe_tree

void attn_tree(const qe_kv_cache_t& c, int layer, const AttnTreeArgs& x, hipStream_t st) {
    CHECK(layer >= 0 && layer < c.layers, "qe_attn_tree: layer %d of %d", layer, c.layers);
    CHECK(x.nseq >= 0 && x.nseq <= kMaxTreeBatch, "qe_attn_tree: nseq = %d (at most %d)", x.nseq, kMaxTreeBatch);
    CHECK(x.t >= 0 && x.t <= kMaxRows && x.max_new >= 1 && x.max_new <= kMaxTreeNodes, "qe_attn_tree: t = %d, max_new = %d (1 .. %d)", x.t, x.max_new, kMaxTreeNodes);
    CHECK(x.scale >= 0x1p-126f && x.scale <= 0x1p126f, "qe_attn_tree: scale %g", (double)x.scale);
    CHECK(x.heads >= c.kv_heads && x.heads % c.kv_heads == 0 && x.heads <= 65535, "qe_attn_tree: %d heads over %d", x.heads, c.kv_heads);
    // units of tokens are counted in 32 bits; no kernel has smaller ones than 128 rows (or all) and 32 tokens
    const int64_t rbs = ((int64_t)x.max_new * (x.heads / c.kv_heads) + 127) / 128, units = ((int64_t)c.width * c.page + 31) / 32;
    CHECK((int64_t)x.nseq * c.kv_heads * rbs <= ((int64_t)1 << 30) / units, "qe_attn_tree: %d sequences x %d heads x %lld blocks of rows x %lld of tokens pass 2^30",
          x.nseq, c.kv_heads, (long long)rbs, (long long)units);
    if (x.nseq == 0 || x.t == 0) return;
    CHECK(x.q && x.out && x.seqs && x.cu, "qe_attn_tree: null pointer");
    CHECK((((uintptr_t)x.q | (uintptr_t)x.out) & 15) == 0 && ((x.q_row | x.q_head | x.o_row | x.o_head) & 7) == 0,
          "qe_attn_tree: q and out must be 16-byte aligned with strides of 8 elements");
    qe_tree::Args a{};
    a.q = (const char*)x.q;
    a.k = (const char*)c.k + 2 * (int64_t)layer * c.layer_stride;
    a.v = (const char*)c.v + 2 * (int64_t)layer * c.layer_stride;
    a.out = (char*)x.out;
    a.lse = x.lse;
    a.q_row = 2 * x.q_row;
    a.q_head = 2 * x.q_head;
    a.o_row = 2 * x.o_row;
    a.o_head = 2 * x.o_head;
    a.page = 2 * c.page_stride;
    a.head = 2 * c.head_stride;
    a.token = 2 * c.token_stride;
    a.table = c.table;
    a.length = c.length;
    a.seqs = x.seqs;
    a.cu = x.cu;
    a.mask = x.mask;
    a.nseq = x.nseq;
    a.t = x.t;
    a.max_new = x.max_new;
    a.heads = x.heads;
    a.kv_heads = c.kv_heads;
    a.group = x.heads / c.kv_heads;
    a.shift = log2_of(c.page);
    a.pages = c.pages;
    a.width = c.width;
    a.slots = c.slots;
    a.scale2 = x.scale * kLog2e;
    if (c.f16) qe_tree::by_shape<kAttnF16>(a, c.d, st);
    else qe_tree::by_shape<kAttnBF16>(a, c.d, st);
}
