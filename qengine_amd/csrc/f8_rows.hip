// Row operators around the 8-bit products (f8.hpp): the norm with the residual's addition, the activation, both quantized to
// e4m3 with a scale for each 128 columns, the sum of the experts' rows, and the weights' layout. All are bound by memory
// for many rows and by the launch for few.
//
// Quantization of a group: a = max |v| (at least 448 * 2^-100, so that a group of zeros has a scale that is a number), scale =
// a / 448, q = e4m3(v * (448 / a)) to nearest even. 448 / a is at most 2^100, |v * (448 / a)| at most 448 (1 + 2^-23), which
// rounds to 448. 16 lanes of 8 columns hold a group, so its maximum takes four lane rotations within a row of 16. An
// infinity makes its group's scale infinite and itself a NaN, a NaN stays in its place: products with either are NaN.
#include "f8.hpp"

namespace {
constexpr float kMax = 448.f;
constexpr float kLeast = 448.f * 7.888609052210118e-31f;  // 2^-100

typedef uint32_t u32x4_f8 __attribute__((ext_vector_type(4)));

template <int T>
__device__ __forceinline__ float get1(const void* p, int64_t i) {
    if constexpr (T == kF8F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (T == kF8BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
    else return f16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void put1(void* p, int64_t i, float v) {
    if constexpr (T == kF8F32) reinterpret_cast<float*>(p)[i] = v;
    else if constexpr (T == kF8BF16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
    else reinterpret_cast<uint16_t*>(p)[i] = f32_to_f16(v);
}
// 8 values from element i on: VEC: 16-byte aligned and all there; else n of them, zeros behind
template <int T, bool VEC>
__device__ __forceinline__ void get8(const void* p, int64_t i, int n, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < n ? get1<T>(p, i + j) : 0.f;
    } else if constexpr (T == kF8F32) {
        const f32x4_v* q = reinterpret_cast<const f32x4_v*>(reinterpret_cast<const float*>(p) + i);
        const f32x4_v a = q[0], b = q[1];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
    } else {
        const u32x4_f8 a = *reinterpret_cast<const u32x4_f8*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t w = a[j];
            if constexpr (T == kF8BF16) {
                v[2 * j] = __uint_as_float(w << 16);
                v[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
            } else {
                v[2 * j] = f16_to_f32((uint16_t)w);
                v[2 * j + 1] = f16_to_f32((uint16_t)(w >> 16));
            }
        }
    }
}
template <int T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return T == kF8BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
template <int T, bool VEC>
__device__ __forceinline__ void put8(void* p, int64_t i, int n, const float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) put1<T>(p, i + j, v[j]);
    } else if constexpr (T == kF8F32) {
        f32x4_v* q = reinterpret_cast<f32x4_v*>(reinterpret_cast<float*>(p) + i);
        q[0] = f32x4_v{v[0], v[1], v[2], v[3]};
        q[1] = f32x4_v{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4_f8*>(reinterpret_cast<uint16_t*>(p) + i) =
            u32x4_f8{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
    }
}
template <int T>
__device__ __forceinline__ float rounded(float v) {
    if constexpr (T == kF8F32) return v;
    else if constexpr (T == kF8BF16) return bf16_to_f32(f32_to_bf16(v));
    else return f16_round(v);
}

template <int ROT>
__device__ __forceinline__ float rot16(float v) {  // the value of the lane ROT places on, in its row of 16
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x120 + ROT, 0xf, 0xf, true));
}
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, rot16<8>(v));
    v = fmaxf(v, rot16<4>(v));
    v = fmaxf(v, rot16<2>(v));
    return fmaxf(v, rot16<1>(v));
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// this lane's 8 of a group that its row of 16 lanes holds: bytes to q (n of them), the scale by the first lane
template <bool VEC>
__device__ __forceinline__ void quantize8(const float (&v)[8], uint8_t* q, int n, float* s, int lane) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 8; j++) a = fmaxf(a, fabsf(v[j]));
    a = fmaxf(max16(a), kLeast);
    const float m = kMax / a;
    const uint2 b = {e4m3x4(v[0] * m, v[1] * m, v[2] * m, v[3] * m), e4m3x4(v[4] * m, v[5] * m, v[6] * m, v[7] * m)};
    if constexpr (VEC) {
        if (n > 0) *reinterpret_cast<uint2*>(q) = b;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) q[j] = (uint8_t)((j < 4 ? b.x : b.y) >> (8 * (j & 3)));
    }
    if ((lane & 15) == 0 && n > 0) *s = a / kMax;
}

// ---------------------------------------------------------------- the norm
// A block holds whole rows, one after another, in registers: NV chunks of 8 columns a thread, as many threads as that takes. The mean is of the rounded
// h, what the residual stream holds. Squares of values past 2^63 leave fp32 in the sum: such a row is summed again with a
// factor of 2^-80, and eps with 2^-160, so every finite row has finite results. Rows beyond 32768 (NV = 8 of 1024 threads) spill 26 to 35
// registers a lane: 1000 rows of 65536 in 77 us, 3.4 TB/s, where 4000 of 16384 run at 4.5.
template <int T, int WT, int NV, bool VEC>
__global__ void __launch_bounds__(1024) norm_kernel(F8Norm a) {
    __shared__ float part[2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, NTH = blockDim.x, waves = NTH >> 6;
    const int chunks = (a.d + 7) >> 3;
    constexpr bool KEEP = NV <= 2;  // the weights for all rows; of long rows they are read again
    float w[KEEP ? NV : 1][8];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = tid + i * NTH;
            if (c < chunks) get8<WT, VEC>(a.w, c * 8, a.d - c * 8, w[i]);
        }
    }
    auto block_sum = [&](float v, int slot) {
#pragma unroll
        for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
        if (waves > 1) {
            if (lane == 0) part[slot][wave] = v;
            __syncthreads();
            v = 0.f;
            for (int i = 0; i < waves; i++) v += part[slot][i];
        }
        return v;
    };
    for (int row = blockIdx.x; row < a.t; row += gridDim.x) {
        float v[NV][8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = tid + i * NTH, n = a.d - c * 8;
            if (c < chunks) {
                get8<T, VEC>(a.x, row * a.ldx + c * 8, n, v[i]);
                if (a.res) {
                    float r[8];
                    get8<T, VEC>(a.res, row * a.ldr + c * 8, n, r);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[i][j] = rounded<T>(v[i][j] + r[j]);
                    put8<T, VEC>(a.res_out, row * a.ldro + c * 8, n, v[i]);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) sum = fmaf(v[i][j], v[i][j], sum);
            }
        }
        sum = block_sum(sum, 0);
        float rs = rsqrtf(sum / a.d + a.eps), half = 1.f;
        if (!(sum <= 3.0e38f)) {  // the same for the whole block
            constexpr float f = 8.271806125530277e-25f;  // 2^-80
            float far = 0.f;
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (tid + i * NTH < chunks) {
#pragma unroll
                    for (int j = 0; j < 8; j++) far = fmaf(v[i][j] * f, v[i][j] * f, far);
                }
            half = 9.094947017729282e-13f;  // 2^-40, for the value and for the root: by all of f small values would lose bits
            rs = rsqrtf(block_sum(far, 1) / a.d + a.eps * f * f) * half;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = tid + i * NTH, n = a.d - c * 8;
            float y[8];
            if (!KEEP && c < chunks) get8<WT, VEC>(a.w, c * 8, n, w[0]);
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = c < chunks ? v[i][j] * half * rs * w[KEEP ? i : 0][j] : 0.f;
            if (a.y && c < chunks) put8<T, VEC>(a.y, row * a.ldy + c * 8, n, y);
            if (a.q)
                quantize8<VEC>(y, reinterpret_cast<uint8_t*>(a.q) + row * a.ldq + c * 8, n, a.s + row * a.s_row + (c >> 4) * a.s_group, lane);
        }
        if (waves > 1) __syncthreads();  // before `part` is written again
    }
}

template <int T, int WT, bool VEC>
void norm_t(const F8Norm& a, hipStream_t st) {
    const unsigned blocks = (unsigned)(a.t < (1 << 20) ? a.t : 1 << 20);
    const int chunks = (a.d + 7) / 8;
#define QE_NORM(NV_) norm_kernel<T, WT, NV_, VEC><<<dim3(blocks), dim3((chunks + NV_ * 64 - 1) / (NV_ * 64) * 64), 0, st>>>(a)
    if (chunks <= 1024) QE_NORM(1);
    else if (chunks <= 2048) QE_NORM(2);
    else if (chunks <= 4096) QE_NORM(4);
    else QE_NORM(8);
#undef QE_NORM
    HIP_CHECK(hipGetLastError());
}
template <int T, int WT>
void norm_v(const F8Norm& a, hipStream_t st) {
    auto al = [](const void* p, int64_t ld, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0 && ld % 8 == 0; };
    const bool vec = a.d % 8 == 0 && al(a.x, a.ldx, 16) && al(a.w, 0, 16) && (!a.res || (al(a.res, a.ldr, 16) && al(a.res_out, a.ldro, 16))) &&
                     (!a.y || al(a.y, a.ldy, 16)) && (!a.q || al(a.q, a.ldq, 8));
    if (vec) norm_t<T, WT, true>(a, st);
    else norm_t<T, WT, false>(a, st);
}

// ---------------------------------------------------------------- quantized rows, silu(gate) * up
// g / (1 + exp(-g)). exp(-g) = 2^t, t = -g log2 e, whose rounding (up to half a step of t, 60 steps of the result) is put back by its
// remainder; where |t| is 126 or more, t may be infinite and e is next to nothing: without it. exp2 and the reciprocal are the hardware's, one step off at most: with
// the library's exp and an IEEE division 4096 x 17408 took 84 us, bound by the vector ALU.
__device__ __forceinline__ float silu(float g) {
    constexpr float L = 1.44269504088896340736f, Lo = 1.92596299112661746887e-08f, ln2 = 0.693147180559945309417f;
    const float t = -g * L, rest = fmaf(-g, Lo, fmaf(-g, L, -t)) * ln2, e = __builtin_amdgcn_exp2f(t);
    return g * __builtin_amdgcn_rcpf(1.f + (fabsf(t) < 126.f ? fmaf(e, rest, e) : e));
}

// silu(g) * u below kFarGate, where 1 + exp(-g) is exp(-g) in fp32, and it or its reciprocal leaves fp32 from -87.3 on: g exp(g) u, the
// exponential as two equal factors, u between them: both are numbers of full precision, and no product leaves fp32, as far as the result is above what a
// group's scale makes zero. The factors' two steps each, the remainder's and three products' roundings: 8 half steps, as above.
constexpr float kFarGate = -40.f;
__device__ __forceinline__ float silu_far(float g, float u) {
    constexpr float L = 1.44269504088896340736f, Lo = 1.92596299112661746887e-08f, ln2 = 0.693147180559945309417f;
    const float t = -g * L, rest = fmaf(-g, Lo, fmaf(-g, L, -t)) * ln2, h = __builtin_amdgcn_exp2f(-0.5f * t);
    return (t < 256.f ? fmaf(g, -rest, g) : g) * h * u * h;
}

// LANES threads a row (a multiple of 16, a power of two), 8 columns each at a time
template <int T, bool GLU, bool VEC>
__global__ void __launch_bounds__(256) act_kernel(F8Act a, int shift, int blocks_a_row) {
    const int lane = threadIdx.x & 63, per = 256 >> shift;
    const int part = blockIdx.x % blocks_a_row;
    const int64_t row = (int64_t)(blockIdx.x / blocks_a_row) * per + (threadIdx.x >> shift);
    const int c = (part << 8) + (threadIdx.x & ((1 << shift) - 1)), n = row < a.t ? a.d - c * 8 : 0;
    float v[8] = {};
    if (n > 0) {
        get8<T, VEC>(a.x, row * a.ldx + c * 8, n, v);
        if constexpr (GLU) {
            float u[8];
            get8<T, VEC>(a.x, row * a.ldx + a.d + c * 8, n, u);
            float least = v[0];
#pragma unroll
            for (int j = 1; j < 8; j++) least = fminf(least, v[j]);
            if (least < kFarGate) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = v[j] < kFarGate ? silu_far(v[j], u[j]) : silu(v[j]) * u[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = silu(v[j]) * u[j];
            }
        }
    }
    quantize8<VEC>(v, reinterpret_cast<uint8_t*>(a.q) + row * a.ldq + c * 8, n, a.s + row * a.s_row + (c >> 4) * a.s_group, lane);
}

template <int T, bool GLU>
void act_t(const F8Act& a, hipStream_t st) {
    const int chunks = (a.d + 7) / 8;
    int shift = 4;
    while (shift < 8 && (1 << shift) < chunks) shift++;
    const int per_row = (chunks + 255) / 256;
    const int64_t blocks = ((int64_t)a.t + (256 >> shift) - 1) / (256 >> shift) * per_row;
    const bool vec = a.d % 8 == 0 && ((uintptr_t)a.x & 15) == 0 && a.ldx % 8 == 0 && ((uintptr_t)a.q & 7) == 0 && a.ldq % 8 == 0;
    if (vec) act_kernel<T, GLU, true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, shift, per_row);
    else act_kernel<T, GLU, false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, shift, per_row);
    HIP_CHECK(hipGetLastError());
}

// ---------------------------------------------------------------- the experts' rows into tokens
// 8 columns of a token a thread, its rows in the order of j: the same sum on every call
template <int T, int OT, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(F8Combine a, int shift, int blocks_a_row) {
    const int per = 256 >> shift, part = blockIdx.x % blocks_a_row;
    const int64_t row = (int64_t)(blockIdx.x / blocks_a_row) * per + (threadIdx.x >> shift);
    const int c = (part << 8) + (threadIdx.x & ((1 << shift) - 1)), n = row < a.t ? a.d - c * 8 : 0;
    if (n <= 0) return;
    float sum[8] = {};
    if (a.add) get8<OT, VEC>(a.add, row * a.ldadd + c * 8, n, sum);
    constexpr int AHEAD = 4;  // rows on their way; each four wait for their indexes first: ten rows of a token are three rounds of index, then row
    for (int j0 = 0; j0 < a.topk; j0 += AHEAD) {
        float v[AHEAD][8], w[AHEAD];
        bool has[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            has[j] = j0 + j < a.topk;
            const int from = has[j] ? a.inv[row * a.topk + j0 + j] : 0;
            w[j] = has[j] ? a.w[row * a.topk + j0 + j] : 0.f;
            has[j] = has[j] && (unsigned)from < (unsigned)a.rows;
            if (has[j]) get8<T, VEC>(a.y, from * a.ldy + c * 8, n, v[j]);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (has[j]) {
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] = fmaf(w[j], v[j][i], sum[i]);
            }
    }
    put8<OT, VEC>(a.out, row * a.ldout + c * 8, n, sum);
}

template <int T, int OT>
void combine_t(const F8Combine& a, hipStream_t st) {
    const int chunks = (a.d + 7) / 8;
    int shift = 4;
    while (shift < 8 && (1 << shift) < chunks) shift++;
    const int per_row = (chunks + 255) / 256;
    const int64_t blocks = ((int64_t)a.t + (256 >> shift) - 1) / (256 >> shift) * per_row;
    auto al = [](const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; };
    const bool vec = a.d % 8 == 0 && al(a.y, a.ldy) && al(a.out, a.ldout) && (!a.add || al(a.add, a.ldadd));
    if (vec) combine_kernel<T, OT, true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, shift, per_row);
    else combine_kernel<T, OT, false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(a, shift, per_row);
    HIP_CHECK(hipGetLastError());
}

// ---------------------------------------------------------------- the weights' layout
__global__ void __launch_bounds__(256) tile_kernel(const uint8_t* __restrict__ src, int64_t ld, int64_t mat, int n, int k, int n16, int kb,
                                                   int64_t total, u32x4_f8* __restrict__ dst) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int in = (int)(i & 127), r = in & 15, chunk = in >> 4;
        const int64_t tile = i >> 7;
        const int b = (int)(tile % kb);
        const int64_t rest = tile / kb;
        const int row = (int)(rest % n16) * 16 + r, at = b * 128 + chunk * 16;
        const int64_t e = rest / n16;
        u32x4_f8 v = {0, 0, 0, 0};
        if (row < n && at < k) v = *reinterpret_cast<const u32x4_f8*>(src + e * mat + row * ld + at);
        dst[i] = v;
    }
}
}  // namespace

void f8_norm(const F8Norm& a, hipStream_t st) {
    CHECK(a.t > 0 && a.t <= kF8MaxRows && a.d > 0 && a.d <= kF8MaxCols, "rms_norm: %d rows of %d", a.t, a.d);
    CHECK(a.x && a.w && (a.y || a.q) && (!a.q || a.s) && !a.res == !a.res_out, "rms_norm: a tensor is missing");
    CHECK(a.eps >= 0x1p-100f && a.eps <= 0x1p100f, "rms_norm: eps %g", (double)a.eps);
#define QE_N(T_) (a.wtype == kF8F32 ? norm_v<T_, kF8F32>(a, st) : norm_v<T_, T_>(a, st))
    if (a.type == kF8BF16) QE_N(kF8BF16);
    else QE_N(kF8F16);
#undef QE_N
}

void f8_act(const F8Act& a, hipStream_t st) {
    CHECK(a.t > 0 && a.t <= kF8MaxRows && a.d > 0 && a.d <= kF8MaxDim, "act_f8: %d rows of %d", a.t, a.d);
    CHECK(a.x && a.q && a.s, "act_f8: a tensor is missing");
    const int64_t blocks = (int64_t)a.t * ((a.d + 2047) / 2048);
    CHECK(blocks <= kF8MaxBlocks * 2, "act_f8: %d rows of %d are too many for a call", a.t, a.d);
    if (a.type == kF8BF16) a.glu ? act_t<kF8BF16, true>(a, st) : act_t<kF8BF16, false>(a, st);
    else a.glu ? act_t<kF8F16, true>(a, st) : act_t<kF8F16, false>(a, st);
}

void f8_combine(const F8Combine& a, hipStream_t st) {
    CHECK(a.t > 0 && a.t <= kF8MaxRows && a.d > 0 && a.d <= kF8MaxDim && a.topk >= 0 && a.topk <= 1024 && a.rows >= 0,
          "moe_combine: %d tokens of %d, %d rows each of %d", a.t, a.d, a.topk, a.rows);
    CHECK(a.out && (a.rows == 0 || a.y) && (a.topk == 0 || (a.inv && a.w)), "moe_combine: a tensor is missing");
    CHECK((int64_t)a.t * ((a.d + 2047) / 2048) <= kF8MaxBlocks * 2, "moe_combine: %d tokens of %d are too many for a call", a.t, a.d);
#define QE_C(T_) (a.otype == kF8F32 ? combine_t<T_, kF8F32>(a, st) : combine_t<T_, T_>(a, st))
    if (a.type == kF8BF16) QE_C(kF8BF16);
    else if (a.type == kF8F16) QE_C(kF8F16);
    else combine_t<kF8F32, kF8F32>(a, st);
#undef QE_C
}

void f8_tile(const void* src, int64_t ld, int64_t mat, int n, int k, int experts, void* dst, hipStream_t st) {
    CHECK(n > 0 && n <= kF8MaxDim && k > 0 && k <= kF8MaxDim && k % 16 == 0 && experts > 0 && experts <= kF8MaxExperts,
          "tile_f8: n = %d, k = %d, %d matrices", n, k, experts);
    CHECK(src && dst && ld % 16 == 0 && mat % 16 == 0 && ((uintptr_t)src & 15) == 0 && ((uintptr_t)dst & 15) == 0, "tile_f8: alignment");
    const int n16 = (n + 15) / 16, kb = (k + 127) / 128;
    const int64_t total = (int64_t)experts * n16 * kb * 128, blocks = (total + 255) / 256;
    tile_kernel<<<dim3((unsigned)(blocks < (1 << 16) ? blocks : 1 << 16)), dim3(256), 0, st>>>(
        static_cast<const uint8_t*>(src), ld, mat, n, k, n16, kb, total, static_cast<u32x4_f8*>(dst));
    HIP_CHECK(hipGetLastError());
}
