// One wave's part of attention with 32 or 64 keys a step in LDS (attn_prompt.hip, attn_wide.hip): 32 query rows with their
// queries, their scores S^T = K Q^T (32 x 32 x 16 MFMA) and their sums O^T = V^T P^T in registers, the running maximum and
// sum of the softmax beside them.
#pragma once
#include "attn_common.hpp"
#include "mfma_tile.hpp"

// Tiles in LDS. A row is CH = D / 8 pieces of 16 bytes, a DMA instruction fills 1 KB = RK rows.
// K: a wave reads one piece of 32 rows (ds_read_b128), so 16 neighbouring rows must have it in 16 different places of a
// 256-byte line: pieces are permuted inside groups of 1, 2 or 4 by row, and each KB starts PAD bytes further on.
// V: a transposing read (ds_read_b64_tr_b16) takes 64 bytes of 8 rows, 4 rows at a time: the 64-byte windows of a row are
// permuted by row.
// Both permutations touch few bits, so a lane's addresses are one to four bases and constants.
template <int D, int KEYS>
struct Tile {
    static constexpr int CH = D / 8, RK = 64 / CH, PAD = D == 256 ? 32 : 64;
    static constexpr int KBYTES = KEYS / RK * (1024 + PAD), VBYTES = KEYS * D * 2, STAGE = KBYTES + VBYTES;
    static __device__ __forceinline__ int kx(int r) { return D == 256 ? r & 1 : D == 128 ? r & 3 : r >> 1 & 3; }
    static __device__ __forceinline__ int vx(int r) { return (D == 64 ? r >> 1 & 1 : r & 3) << 2; }
    static __device__ __forceinline__ int k_row(int r) { return r / RK * (1024 + PAD) + r % RK * (D * 2); }
};

template <int DT, int D, int KEYS>
struct Wave32 {
    using T = AttnT<DT>;
    using L = Tile<D, KEYS>;
    static constexpr int KS = D / 16, DB = D / 32, NX = KEYS / 32;
    struct Scores {
        f32x16_v s[NX];  // keys 32 x + 8 (e / 4) + 4 (lane / 32) + e % 4 of a step
    };
    u32x4_v q[KS];  // lane: query lane % 32, values 16 ks + 8 (lane / 32) ..
    f32x16_v o[DB]; // lane: query lane % 32, columns 32 db + 8 (e / 4) + 4 (lane / 32) + e % 4
    float m, l;     // maximum (times the scale, base 2) and this half's sum
    float lazy;     // kLazy, or -inf once a row of the wave has its maximum beyond kFar
    // the lane's places in a K tile (row lane % 32, piece 2 ks + lane / 32 for ks = 0 and 1) and in a V tile (row 4 (lane /
    // 32) + (0 .. 3) by lane, columns 32 d + 16 (lane / 16 % 2) + 4 (lane % 4) for d = 0 .. 3)
    int kat[2], vat[4];

    __device__ __forceinline__ void places(int lane) {
        const int col = lane & 31, half = lane >> 5, vr = 4 * half + (lane & 15) / 4, vc = (lane >> 4 & 1) * 2 + (lane & 3) / 2;
#pragma unroll
        for (int i = 0; i < 2; i++) kat[i] = L::k_row(col) + (((2 * i + half) ^ L::kx(col)) * 16);
#pragma unroll
        for (int d = 0; d < 4; d++) vat[d] = L::KBYTES + vr * D * 2 + (((4 * d + vc) ^ L::vx(vr)) * 16) + (lane & 1) * 8;
    }
    // row: the lane's query
    __device__ __forceinline__ void load_queries(const char* row, int half) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] = *reinterpret_cast<const u32x4_v*>(row + half * 16 + ks * 32);
    }
    // The queries are waited for here: a use inside the loop would make the compiler wait there for whatever loads are in
    // flight, which are the next steps'.
    __device__ __forceinline__ void await_queries() {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(q[ks]));
    }
    __device__ __forceinline__ void clear() {
        m = kNegInf;
        l = 0.f;
        lazy = kLazy;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.f;
    }
    // Scores of a step. seen(x, e): whether the lane's query sees the key of s[x][e] (asked if masked). Operands are read in
    // groups, a group ahead of the products that use it.
    template <class Seen>
    __device__ __forceinline__ Scores scores(const char* tile, bool masked, Seen seen) const {
        Scores r;
        f32x16_v(&s)[NX] = r.s;
        constexpr int GK = D == 256 ? 4 : NX == 1 ? 2 : 8, NK = NX * KS / GK;
        u32x4_v kf[2][GK];
        auto read_k = [&](int g) {
#pragma unroll
            for (int i = 0; i < GK; i++) {
                const int x = (g * GK + i) % NX, ks = (g * GK + i) / NX;
                constexpr int M = D == 256 ? 1 : 2;  // bases
                const int at = kat[ks % M] + ks / M * M * 32 + 32 / L::RK * (1024 + L::PAD) * x;
                kf[g % 2][i] = *reinterpret_cast<const u32x4_v*>(tile + at);
            }
        };
#pragma unroll
        for (int x = 0; x < NX; x++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[x][e] = 0.f;
        read_k(0);
#pragma unroll
        for (int g = 0; g < NK; g++) {
            if (g + 1 < NK) read_k(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < GK; i++) s[(g * GK + i) % NX] = T::mfma32(kf[g % 2][i], q[(g * GK + i) / NX], s[(g * GK + i) % NX]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (masked) {
#pragma unroll
            for (int x = 0; x < NX; x++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    s[x][e] = seen(x, e) ? s[x][e] : kNegInf;
        }
        return r;
    }
    // Softmax of the scores and their products with the step's values, whose first reads are under way during the softmax
    __device__ __forceinline__ void values(const char* tile, Scores r, int pass, float scale2) {
        f32x16_v(&s)[NX] = r.s;
        constexpr int GV = NX == 1 ? 2 : 4, NV = DB * 2 * NX / GV;
        u32x4_v vf[2][GV];
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
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        float mx = kNegInf;
#pragma unroll
        for (int x = 0; x < NX; x++) {
            if constexpr (D == 256) asm("" : "+v"(s[x]));  // not in accumulators, from where each use below would read them
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[x][e]);
        }
        mx = __builtin_fmaf(mx, scale2, pass == 1 ? T::kRoom : 0.f);
        float less = m == kNegInf ? 0.f : m;
        if (__any(mx - m > lazy)) {  // (m + kLazy would round up to the next number where that is 2 kLazy away)
            const float top = fmaxf(m, max_over_halves(mx));
            const float f0 = top == kNegInf || pass > 1 ? 1.f : __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= f0;
#pragma unroll
            for (int d = 0; d < DB; d++) o[d] *= f0;
            less = m == kNegInf ? 0.f : m;
            if (pass <= 1 && __any(fabsf(less) > kFar)) {  // this step's exponents, and from now on every step's
                lazy = kNegInf;
#pragma unroll
                for (int x = 0; x < NX; x++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[x][e] = mul_rounded(s[x][e], scale2) - less;
                scale2 = 1.f;
                less = 0.f;
                asm volatile("" : "+s"(scale2), "+v"(less));  // no copy of the products below for these constants
            }
        }
        // rounded to the values' type, since the matrix cores take nothing wider at that rate; their sum is not
        u32x4_v p[2 * NX];
#pragma unroll
        for (int x = 0; x < NX; x++)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], scale2, -less));
                const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e + 1], scale2, -less));
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
    // After the steps: the sums as they are. (Without it the compiler keeps a second copy of them in the order of the stores
    // that follow and moves all of them at every step.)
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int d = 0; d < DB; d++) asm volatile("" : "+v"(o[d]));
    }
    // The sums of `groups` waves with the same rows into the first one's, through LDS: every lane's partner holds the same
    // rows and columns. Every wave of the block calls it.
    static constexpr int group_bytes(int waves, int groups) { return (groups - 1) * waves * (DB * 16 + 2) * 256; }
    __device__ __forceinline__ void add_groups(float* lds, int wave, int group, int waves, int groups, int lane, int pass) {
        __syncthreads();  // all are done with the stages
        auto at = [&](int g, int i) { return lds + (((g - 1) * waves + wave) * (DB * 16 + 2) + i) * 64 + lane; };
        if (group > 0) {
            *at(group, 0) = m;
            *at(group, 1) = l;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) *at(group, 2 + d * 16 + e) = o[d][e];
        }
        __syncthreads();
        if (group == 0) {
            float top = m;
            for (int g = 1; g < groups; g++) top = fmaxf(top, *at(g, 0));
            for (int g = 0; g < groups; g++) {
                const float mg = g ? *at(g, 0) : m;
                float f = mg == kNegInf ? 0.f : __builtin_amdgcn_exp2f(mg - top);
                if (mg == __builtin_huge_valf() || pass > 1) f = 1.f;  // (a row with such a maximum is NaN already)
                if (g == 0) {
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DB; d++) o[d] *= f;
                } else {
                    l += f * *at(g, 1);
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[d][e] += f * *at(g, 2 + d * 16 + e);
                }
            }
            m = top;
        }
    }
    // whether a sum is not finite, or about not to be
    __device__ __forceinline__ bool bad() const {
        float x = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) x = if_bad(o[d][e], x);
        return !(x == 0.f);
    }
    // out: column 4 (lane / 32) of the lane's row; l: the whole row's sum
    __device__ __forceinline__ void store(char* out, float inv) const {
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                uint2 w;
                w.x = T::pack(o[d][e] * inv, o[d][e + 1] * inv);
                w.y = T::pack(o[d][e + 2] * inv, o[d][e + 3] * inv);
                *reinterpret_cast<uint2*>(out + d * 64 + e * 4) = w;
            }
    }
    // after a pass over one kind of values: the outputs that see one
    __device__ __forceinline__ void store_kind(char* out, int pass) const {
#pragma unroll
        for (int d = 0; d < DB; d++) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                uint16_t* at = reinterpret_cast<uint16_t*>(out + d * 64 + e / 4 * 16 + e % 4 * 2);
                const uint16_t was = *at;
                *at = o[d][e] > 0.f ? add_kind<DT>(was, pass) : was;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the same for sums in 32 bits
    __device__ __forceinline__ void store_kind(float* sums, int pass) const {
#pragma unroll
        for (int d = 0; d < DB; d++) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float* at = sums + d * 32 + e / 4 * 8 + e % 4;
                const float was = *at, now = pass == 2 ? was + __builtin_huge_valf() : pass == 3 ? was - __builtin_huge_valf() : __builtin_nanf("");
                *at = o[d][e] > 0.f ? now : was;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};
