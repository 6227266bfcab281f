// What the two kernels of attention over the cache share (attn_tree.hip: few rows of a kv head, attn_wide.hip: more): their
// arguments, how work is split, and the launch that joins the parts.
//
// Unit: UNIT tokens of one (sequence, kv head, block of ROWS rows); a row is a drafted token times a query head of the kv
// head's group. The units in that order are dealt to as many blocks as the device holds, in ranges of equal length, whatever
// the sequences' lengths. A (sequence, head, row block) that ends up in several blocks leaves partial sums (fp32, with their
// running maximum and sum) in a workspace, which join_kernel adds in block order.
#pragma once
#include "attn_common.hpp"
#include "kv_cache.hpp"

#include <algorithm>

namespace qe_tree {
constexpr int kThreads = 256;

struct Args {
    const char *q, *k, *v;
    char* out;
    float* lse;
    int64_t q_row, q_head, o_row, o_head, page, head, token;  // bytes
    const int32_t *table, *length, *seqs, *cu;
    const uint64_t* mask;
    int nseq, t, max_new, heads, kv_heads, group, shift, pages, width, slots, rb_max;
    float scale2;  // log2(e) times the scale: exponentials are powers of two
    float* part;   // [block][2][rows][D] partial sums, nullptr: every block takes whole (sequence, head, row block)s
    float2* ml;    // [block][2][rows] maximum and sum
    int* ends;     // [nseq] end of each sequence's units, then the range length
};

struct Seq {
    int first, n, len, total;  // first row, rows, committed tokens, all tokens
    int slot;
};
__device__ __forceinline__ Seq seq_of(const Args& a, int b) {
    Seq s;
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    s.first = min(max(c0, 0), a.t);
    s.n = min(min(c1, a.t) - s.first, a.max_new);
    s.slot = a.seqs[b];
    const bool ok = s.slot >= 0 && s.slot < a.slots;
    const int room = a.width << a.shift;
    s.len = ok ? min(max(a.length[ok ? s.slot : 0], 0), room) : 0;
    s.total = ok ? min(s.len + max(s.n, 0), room) : 0;
    return s;
}
template <int ROWS>
__device__ __forceinline__ int row_blocks(const Args& a, int n) {
    return (n * a.group + ROWS - 1) / ROWS;
}
template <int UNIT>
__device__ __forceinline__ int unit_count(int total) {
    return max(1, (total + UNIT - 1) / UNIT);
}

// The block's units [u, u_end), the sequence of the first and that sequence's first unit; false: none. Every thread of the
// block calls it; ends (nseq ints of LDS) and tmp are free afterwards.
template <int UNIT, int ROWS, int THREADS>
__device__ __forceinline__ bool my_units(const Args& a, int* ends, int* tmp, int& u, int& u_end, int& b, int& base) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (!a.part) {  // a (sequence, head, row block) a block
        u = base = 0;
        u_end = 1;
        b = blockIdx.x / (a.kv_heads * a.rb_max);
        return true;
    }
    int carry = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += THREADS) {
        int x = 0;
        if (b0 + tid < a.nseq) {
            const Seq s = seq_of(a, b0 + tid);
            if (s.n > 0) x = unit_count<UNIT>(s.total) * row_blocks<ROWS>(a, s.n) * a.kv_heads;
        }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) tmp[wave] = x;
        __syncthreads();
        for (int w = 0; w < THREADS / 64; w++)
            if (w < wave) x += tmp[w];
        if (b0 + tid < a.nseq) ends[b0 + tid] = carry + x;
        for (int w = 0; w < THREADS / 64; w++) carry += tmp[w];
    }
    __syncthreads();
    const int range = (carry + gridDim.x - 1) / gridDim.x;
    if (blockIdx.x == 0) {
        for (int i = tid; i < a.nseq; i += THREADS) a.ends[i] = ends[i];
        if (tid == 0) a.ends[a.nseq] = range;
    }
    u = blockIdx.x * range;
    u_end = min(carry, u + range);
    if (u >= u_end) return false;
    int lo = 0, hi = a.nseq - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ends[mid] > u) hi = mid;
        else lo = mid + 1;
    }
    b = lo;
    base = lo > 0 ? ends[lo - 1] : 0;
    __syncthreads();
    return true;
}
// Units [t0, t1), of `units` in all, of the (head, row block) that unit u of a sequence begins; false: no such row block
struct Run {
    int h, rb, t0, t1;
};
__device__ __forceinline__ bool run_of(const Args& a, int base, int u, int u_end, int units, int rbs, Run& r) {
    if (a.part) {
        const int v = u - base;
        r.t0 = v % units;
        r.rb = v / units % rbs;
        r.h = v / units / rbs;
        r.t1 = min(units, r.t0 + u_end - u);
    } else {
        const int v = blockIdx.x % (a.kv_heads * a.rb_max);
        r.h = v / a.rb_max;
        r.rb = v % a.rb_max;
        r.t0 = 0;
        r.t1 = units;
    }
    r.h = __builtin_amdgcn_readfirstlane(r.h);
    r.rb = __builtin_amdgcn_readfirstlane(r.rb);
    r.t0 = __builtin_amdgcn_readfirstlane(r.t0);
    r.t1 = __builtin_amdgcn_readfirstlane(r.t1);
    return r.rb < rbs;
}


// Joins the parts of one row: block (row, kv head, sequence). Four waves take every fourth part; sums in a fixed order.
template <int DT, int D, int ROWS>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a, int most) {
    using T = AttnT<DT>;
    constexpr int E = D / 64, kWaves = kThreads / 64;
    const int r = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c0 = a.cu[b], first = min(max(c0, 0), a.t), n = min(min(a.cu[b + 1], a.t) - first, a.max_new);
    if (r >= n * a.group) return;
    const int u0 = b > 0 ? a.ends[b - 1] : 0, range = a.ends[a.nseq], rbs = row_blocks<ROWS>(a, n), rb = r / ROWS;
    const int units = (a.ends[b] - u0) / (rbs * a.kv_heads);
    const int v0 = u0 + (h * rbs + rb) * units, w0 = v0 / range, w1 = (v0 + units - 1) / range, cnt = w1 - w0 + 1;
    if (cnt == 1) return;
    extern __shared__ float wgt[];  // [most] weights, then the waves' sums
    float* acc = wgt + most;
    __shared__ float red[2][kWaves];
    auto at = [&](int i) { return ((int64_t)(w0 + i) * 2 + (i > 0 ? 0 : 1)) * ROWS + r % ROWS; };
    float top = kNegInf;
    for (int i = tid; i < cnt; i += kThreads) top = fmaxf(top, a.ml[at(i)].x);
#pragma unroll
    for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, red[0][w]);
    float sum = 0.f;
    for (int i = tid; i < cnt; i += kThreads) {
        const float2 x = a.ml[at(i)];
        float f = x.x == kNegInf ? 0.f : __builtin_amdgcn_exp2f(x.x - top);
        if (x.x == __builtin_huge_valf()) f = 1.f;
        wgt[i] = f;
        sum += f * x.y;
    }
#pragma unroll
    for (int o = 32; o; o /= 2) sum += __shfl_xor(sum, o);
    if (lane == 0) red[1][wave] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) sum += red[1][w];
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = 0.f;
#pragma unroll 4
    for (int i = wave; i < cnt; i += kWaves) {
        const float f = wgt[i];
        const float* p = a.part + at(i) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) y[e] += f * p[e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) acc[wave * D + lane * E + e] = y[e];
    __syncthreads();
    const int i = r / a.group, hq = h * a.group + r % a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (tid < D / 2) {
        float z0 = 0.f, z1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            z0 += acc[w * D + 2 * tid];
            z1 += acc[w * D + 2 * tid + 1];
        }
        *reinterpret_cast<uint32_t*>(a.out + (int64_t)(first + i) * a.o_row + (int64_t)hq * a.o_head + 4 * tid) = T::pack(z0 * inv, z1 * inv);
    }
    if (a.lse && tid == 0) a.lse[(int64_t)(first + i) * a.heads + hq] = sum == 0.f ? kNegInf : (top + log2f(sum)) * kLn2;
}

// kernel and join on the stream, or the kernel alone with a (sequence, head, row block) a block where the device has no
// memory for the parts. per_cu: blocks that a CU holds
template <int DT, int D, int UNIT, int ROWS, class Kernel>
void launch_split(Args a, Kernel kernel, int threads, size_t lds, int per_cu, hipStream_t st) {
    a.rb_max = (a.max_new * a.group + ROWS - 1) / ROWS;
    const int64_t runs = (int64_t)a.nseq * a.kv_heads * a.rb_max;
    const int64_t most_units = ((int64_t)(a.width << a.shift) + UNIT - 1) / UNIT;
    CHECK(runs * most_units < (int64_t)1 << 31, "qe_attn_tree: %lld rows x %lld units of tokens", (long long)runs, (long long)most_units);
    const int grid = (int)std::min<int64_t>(runs * most_units, per_cu * qe_num_cus());
    const size_t part = (size_t)grid * 2 * ROWS * D * 4, ml = (size_t)grid * 2 * ROWS * 8, ends = ((size_t)a.nseq + 1) * 4;
    WsHold hold(st);
    if (char* ws = static_cast<char*>(hold.get(kWsAttn, part + ml + ends))) {
        a.part = reinterpret_cast<float*>(ws);
        a.ml = reinterpret_cast<float2*>(ws + part);
        a.ends = reinterpret_cast<int*>(ws + part + ml);
        kernel<<<grid, threads, lds, st>>>(a);
        HIP_CHECK(hipGetLastError());
        join_kernel<DT, D, ROWS><<<dim3(a.max_new * a.group, a.kv_heads, a.nseq), kThreads, (grid + kThreads / 64 * D) * 4, st>>>(a, grid);
    } else {
        kernel<<<(int)runs, threads, lds, st>>>(a);
    }
    HIP_CHECK(hipGetLastError());
}

void attend_wide(const Args& a, int d, bool f16, hipStream_t st);  // attn_wide.hip: any number of rows
}  // namespace qe_tree
