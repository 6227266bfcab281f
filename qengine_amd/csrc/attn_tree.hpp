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
#include "seq_rows.hpp"

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
    const RowRange r = rows_of(a.cu[b], a.cu[b + 1], a.t);
    s.first = r.first;
    s.n = min(r.n, a.max_new);
    s.slot = a.seqs[b];
    const bool ok = s.slot >= 0 && s.slot < a.slots;
    const int room = a.width << a.shift;
    s.len = ok ? min(max(a.length[ok ? s.slot : 0], 0), room) : 0;
    s.total = ok ? min(s.len + s.n, room) : 0;
    return s;
}
// What a block keeps of the sequences of a call with up to kKept of them, so that it does not read them again (three
// dependent reads) for every run that it begins.
constexpr int kKept = 256;
struct Kept {
    Seq seq[kKept];
    int tmp[16];
};
__device__ __forceinline__ Seq seq_at(const Args& a, const Kept& kept, int b) {
    if (!a.part || a.nseq > kKept) return seq_of(a, b);
    return kept.seq[b];
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
// block calls it; ends (nseq ints of LDS) is free afterwards.
template <int UNIT, int ROWS, int THREADS>
__device__ __forceinline__ bool my_units(const Args& a, int* ends, Kept& kept, int& u, int& u_end, int& b, int& base) {
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
            if (b0 + tid < kKept) kept.seq[b0 + tid] = s;
            if (s.n > 0) x = unit_count<UNIT>(s.total) * row_blocks<ROWS>(a, s.n) * a.kv_heads;
        }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) kept.tmp[wave] = x;
        __syncthreads();
        for (int w = 0; w < THREADS / 64; w++)
            if (w < wave) x += kept.tmp[w];
        if (b0 + tid < a.nseq) ends[b0 + tid] = carry + x;
        for (int w = 0; w < THREADS / 64; w++) carry += kept.tmp[w];
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


// Joins the parts of the rows, WPR waves a row, each every WPR-th part; sums in a fixed order. One wave a row where there are
// rows enough to fill the device: with four, 15360 rows of four parts took 21 us.
template <int DT, int D, int ROWS, int WPR>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a, int most) {
    using T = AttnT<DT>;
    constexpr int E = D / 64, RPB = kThreads / 64 / WPR;  // columns of a lane, rows of a block
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave % WPR;
    const int r = blockIdx.x * RPB + wave / WPR, h = blockIdx.y, b = blockIdx.z;
    const RowRange seq = rows_of(a.cu[b], a.cu[b + 1], a.t);
    const int first = seq.first, n = min(seq.n, a.max_new);
    int cnt = 0, w0 = 0;
    if (r < n * a.group) {
        const int u0 = b > 0 ? a.ends[b - 1] : 0, range = a.ends[a.nseq], rbs = row_blocks<ROWS>(a, n);
        const int units = (a.ends[b] - u0) / (rbs * a.kv_heads), v0 = u0 + (h * rbs + r / ROWS) * units;
        w0 = v0 / range;
        cnt = (v0 + units - 1) / range - w0 + 1;
    }
    if (WPR > 1 && cnt < 2) return;  // the whole block: one row
    extern __shared__ float join_lds[];
    float* wgt = join_lds + (WPR > 1 ? 0 : wave * most);  // [most] weights of the parts, and the waves' sums
    float* acc = join_lds + most;
    __shared__ float red[2][kThreads / 64];
    auto at = [&](int i) { return ((int64_t)(w0 + i) * 2 + (i > 0 ? 0 : 1)) * ROWS + r % ROWS; };
    float top = kNegInf, sum = 0.f;
    for (int i = wr * 64 + lane; i < cnt; i += WPR * 64) top = fmaxf(top, a.ml[at(i)].x);
#pragma unroll
    for (int o = 32; o; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    if constexpr (WPR > 1) {
        if (lane == 0) red[0][wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; w++) top = fmaxf(top, red[0][w]);
    }
    for (int i = wr * 64 + lane; i < cnt; i += WPR * 64) {
        const float2 x = a.ml[at(i)];
        float f = x.x == kNegInf ? 0.f : __builtin_amdgcn_exp2f(x.x - top);
        if (x.x == __builtin_huge_valf()) f = 1.f;
        wgt[i] = x.x == kNegInf ? 0.f : above_zero(f);
        sum += f * x.y;
    }
#pragma unroll
    for (int o = 32; o; o /= 2) sum += __shfl_xor(sum, o);
    if (WPR > 1 && lane == 0) red[1][wave] = sum;
    __syncthreads();
    if constexpr (WPR > 1) {
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; w++) sum += red[1][w];
    }
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = 0.f;
#pragma unroll 4
    for (int i = wr; i < cnt; i += WPR) {
        const float f = wgt[i];
        const float* p = a.part + at(i) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) y[e] += f * p[e];
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int e = 0; e < E; e++) acc[wave * D + lane * E + e] = y[e];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int e = 0; e < E; e++) {
            y[e] = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; w++) y[e] += acc[w * D + lane * E + e];
        }
    }
    if (cnt < 2) return;
    const int i = r / a.group, hq = h * a.group + r % a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    char* p = a.out + (int64_t)(first + i) * a.o_row + (int64_t)hq * a.o_head + lane * E * 2;
    if constexpr (E == 1) *reinterpret_cast<uint16_t*>(p) = (uint16_t)T::pack(y[0] * inv, 0.f);
    else if constexpr (E == 2) *reinterpret_cast<uint32_t*>(p) = T::pack(y[0] * inv, y[1] * inv);
    else *reinterpret_cast<uint2*>(p) = make_uint2(T::pack(y[0] * inv, y[1] * inv), T::pack(y[2] * inv, y[3] * inv));
    if (a.lse && lane == 0) a.lse[(int64_t)(first + i) * a.heads + hq] = sum == 0.f ? kNegInf : (top + log2f(sum)) * kLn2;
}

// kernel and join on the stream, or the kernel alone with a (sequence, head, row block) a block where the device has no
// memory for the parts. per_cu: blocks that a CU holds
template <int DT, int D, int UNIT, int ROWS, class Kernel>
void launch_split(Args a, Kernel kernel, int threads, size_t lds, int per_cu, hipStream_t st) {
    a.rb_max = (a.max_new * a.group + ROWS - 1) / ROWS;
    const int64_t runs = (int64_t)a.nseq * a.kv_heads * a.rb_max;
    const int64_t most_units = ((int64_t)(a.width << a.shift) + UNIT - 1) / UNIT;
    const int grid = (int)std::min<int64_t>(runs * most_units, per_cu * qe_num_cus());
    // the same for every call of a kernel, whatever its batch and grid: a stream's buffer is allocated by its first call and
    // kept, not replaced (a hipMalloc and a wait for the stream) by each batch that is larger than those before
    const size_t blocks = (size_t)per_cu * qe_num_cus();
    const size_t part = blocks * 2 * ROWS * D * 4, ml = blocks * 2 * ROWS * 8, ends = ((size_t)kMaxTreeBatch + 1) * 4;
    WsHold hold(st);
    if (char* ws = attn_tree_split() ? static_cast<char*>(hold.get(kWsAttn, part + ml + ends)) : nullptr) {
        a.part = reinterpret_cast<float*>(ws);
        a.ml = reinterpret_cast<float2*>(ws + part);
        a.ends = reinterpret_cast<int*>(ws + part + ml);
        kernel<<<grid, threads, lds, st>>>(a);
        HIP_CHECK(hipGetLastError());
        const int rows = a.max_new * a.group;
        if ((int64_t)rows * a.kv_heads * a.nseq >= 8 * qe_num_cus())
            join_kernel<DT, D, ROWS, 1><<<dim3((rows + 3) / 4, a.kv_heads, a.nseq), kThreads, 4 * grid * 4, st>>>(a, grid);
        else
            join_kernel<DT, D, ROWS, 4><<<dim3(rows, a.kv_heads, a.nseq), kThreads, (grid + 4 * D) * 4, st>>>(a, grid);
    } else {
        kernel<<<(int)runs, threads, lds, st>>>(a);
    }
    HIP_CHECK(hipGetLastError());
}

void attend_wide(const Args& a, int d, bool f16, hipStream_t st);  // attn_wide.hip: any number of rows
}  // namespace qe_tree
