// Operators in 8-bit floating point (e4m3 as OCP defines it: largest value 448, no infinities) and what stands between them
// in a layer: host interface and the parts that the kernels share (f8_rows.hip, f8_dec.hip,
// f8_ring.hip, f8_gemm.hip; f8_matmul.cpp and f8_choice.hpp choose).
//
// Weights [n][k] have one fp32 scale for each block of 128 x 128, activations one for each row's 128 columns; the last block or
// group may be shorter. y[t][n] = sum over blocks b of k: sx[t][b] sw[n / 128][b] (sum over k in b: x[t][k] W[n][k]). The inner
// sum is one MFMA of depth 128 from zero; the outer is an fp32 FMA on the vector ALU.
// What the matrix cores sum: products of 8 consecutive k are aligned to the largest exponent among them and cut at 2^-13 of it
// (measured: 1 and 2^-13 add, 2^-14 is lost; at 8 k or more apart 2^-23 is kept); these sums and the accumulator add as
// fp32. Normally distributed rows: 1.4e-5 of the result's norm, the same for every e4m3 MFMA of this chip. An output of 16 bits (half
// a step: 2^-12 to 2^-8) does not show it, an fp32 output would promise bits that are not there: products are bf16 or fp16.
//
// Weight layout (tile_f8), per matrix: [ceil(n / 16)][ceil(k / 128)][8 chunks of 16 k][16 rows][16 bytes], zeros past n and
// k. A tile of 16 rows x 128 k is 2 KB in one piece, and lane l = 16 g + r of v_mfma_f32_16x16x128_f8f6f4 holds row r's
// chunks g and 4 + g: two loads of 1 KB a wave, every byte of which is used. Which k the matrix core takes for which byte does
// not matter as long as both operands have the same; activations are read by the same chunks.
#pragma once
#include "qe_api.hpp"

enum F8Type : int { kF8F32 = 0, kF8BF16 = 1, kF8F16 = 2 };  // types of outputs, and of the row operators' inputs

struct F8Norm {  // y = h rsqrt(mean(h^2) + eps) w of h = x + res (or x); any of y and q
    const void *x, *res, *w;
    void *res_out, *y, *q;
    float* s;
    int64_t ldx, ldr, ldro, ldy, ldq, s_row, s_group;
    int t, d, type, wtype;
    float eps;
};
struct F8Act {  // rows, or silu(gate) * up of rows [gate d][up d], quantized
    const void* x;
    void* q;
    float* s;
    int64_t ldx, ldq, s_row, s_group;
    int t, d, type;
    bool glu;
};
struct F8Combine {  // out[t] = add[t] + sum_j w[t][j] y[inv[t topk + j]]
    const void *y, *add;
    const int32_t* inv;
    const float* w;
    void* out;
    int64_t ldy, ldadd, ldout;
    int t, topk, rows, d, type, otype;
};
struct F8Mat {  // one product, or (off) one for each segment of rows with its own matrix
    const void* q;
    const float* s;
    const void* x;
    const float* xs;
    const int32_t *off, *rows;
    void* y;
    int64_t ldx, xs_row, xs_group, ldy;
    int n, k, t, r, experts, out;  // t: rows of x, r: of y
};
constexpr int kF8MaxExperts = 1024;
constexpr int kF8MaxCols = 65536;       // of a norm's row
constexpr int kF8MaxDim = 1 << 20;      // n and k
constexpr int kF8MaxRows = 1 << 24;     // of a call
constexpr int kF8MaxRowBytes = 1 << 24;  // from a row of x to the next
constexpr int kF8MaxScaleStride = 1 << 22;  // elements from a row's scale to the next
constexpr int64_t kF8MaxBlocks = 1 << 22;  // of 512 threads: a launch takes less than 2^32 threads

void f8_norm(const F8Norm& a, hipStream_t st);
void f8_act(const F8Act& a, hipStream_t st);
void f8_combine(const F8Combine& a, hipStream_t st);
void f8_tile(const void* src, int64_t ld, int64_t mat, int n, int k, int experts, void* dst, hipStream_t st);
void f8_matmul(const F8Mat& a, hipStream_t st);
void f8_matmul_choice(const F8Mat& a, int bt, int bw, int parts, hipStream_t st);  // bt 16: f8_dec, 256: f8_gemm
void f8_grouped_choice(const F8Mat& a, int bt, hipStream_t st);  // the same, 64 and 128: f8_ring
void f8_dec(const F8Mat& a, hipStream_t st);  // up to 16 rows, or segments of few
void f8_ring(const F8Mat& a, int bt, int bw, int parts, hipStream_t st);  // blocks of bt rows x bw weight rows, K in ranges
void f8_gemm(const F8Mat& a, int parts, hipStream_t st);                  // tiles of 256 x 256
bool f8_gemm_takes(const F8Mat& a);

#ifdef __HIPCC__
typedef int i32x4_f8 __attribute__((ext_vector_type(4)));
typedef int i32x8_f8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8_f8 f8_join(i32x4_f8 lo, i32x4_f8 hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
// D[weight row][token] of 16 x 16, 128 deep: lane l has token l % 16, weight rows 4 (l / 16) + 0..3
__device__ __forceinline__ f32x4_v f8_mfma(i32x8_f8 w, i32x8_f8 x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4_v{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// four consecutive columns of y from column c on; vec: the row's 4-column pieces are aligned
template <int OUT>
__device__ __forceinline__ void f8_store4(uint16_t* row, int c, int n, f32x4_v v, bool vec) {
    if (vec && c + 4 <= n) {
        *reinterpret_cast<uint2*>(row + c) = OUT == kF8BF16 ? uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}
                                                            : uint2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c + i < n) row[c + i] = OUT == kF8BF16 ? f32_to_bf16(v[i]) : f32_to_f16(v[i]);
    }
}
inline bool f8_vec_ok(const void* y, int64_t ldy) { return ldy % 4 == 0 && ((uintptr_t)y & 7) == 0; }

// Segments of experts in blocks of bt rows, shared out evenly in `ways` runs: number `idx` of run `way` -> expert, first row, rows of
// it, or false: there are not so many (a launch has blocks for the most there can be). Every thread of the block
// calls it; sh: NTH / 64 + 4 ints of LDS, free again after the next barrier. Entries of `off` are taken as
// rows in [0, r], segments that do not ascend as empty, so no answer names a row outside.
template <int NTH>
__device__ __forceinline__ bool f8_job(const int32_t* __restrict__ off, int experts, int r, int bt, int way, int ways, int idx, int* sh,
                                       int& e, int& row0, int& rows) {
    constexpr int NWV = NTH / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (experts + NTH - 1) / NTH, first = tid * per;
    auto at = [&](int i) { return min(max(off[min(i, experts)], 0), r); };
    int mine = 0, prev = at(first);
    for (int i = 0; i < per; i++) {
        const int next = at(first + i + 1);
        mine += (max(next - prev, 0) + bt - 1) / bt;
        prev = next;
    }
    int sum = mine;  // of the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(sum, d);
        if (lane >= d) sum += v;
    }
    if (lane == 63) sh[wave] = sum;
    if (tid == 0) sh[NWV] = -1;
    __syncthreads();
    int before = sum - mine, total = 0;
    for (int w = 0; w < NWV; w++) {
        if (w < wave) before += sh[w];
        total += sh[w];
    }
    const int share = (total + ways - 1) / ways, job = idx < share ? way * share + idx : total;
    if (job >= before && job < before + mine) {
        int j = job - before;
        prev = at(first);
        for (int i = 0; i < per; i++) {
            const int next = at(first + i + 1), len = max(next - prev, 0), n = (len + bt - 1) / bt;
            if (j >= 0 && j < n) {
                sh[NWV] = first + i;
                sh[NWV + 1] = prev + j * bt;
                sh[NWV + 2] = min(bt, len - j * bt);
            }
            j -= n;
            prev = next;
        }
    }
    __syncthreads();
    e = __builtin_amdgcn_readfirstlane(sh[NWV]);
    row0 = __builtin_amdgcn_readfirstlane(sh[NWV + 1]);
    rows = __builtin_amdgcn_readfirstlane(sh[NWV + 2]);
    return e >= 0;
}
#endif
inline int64_t f8_most_jobs(int64_t r, int64_t experts, int bt) { return r / bt + (r < experts ? r : experts); }
