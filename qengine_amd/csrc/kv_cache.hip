// The paged cache's own operations: pages given out, shared and given back (one number per page says how many slots hold
// it), rows appended, and the rows of an accepted path moved together. All state is on the device; no call waits for it.
#include "kv_cache.hpp"

#include <algorithm>

namespace {
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256;
constexpr int kOne = 1024;  // threads of the one-block kernel
constexpr int kList = 4096;  // pages that it hands out at a time

struct Pool {
    char *k, *v;
    int64_t layer, page, head, token;  // strides in bytes
    int layers, pages, shift, heads, d;
};
struct Slots {
    int32_t *table, *length, *held, *ref;
    int slots, width, pages, shift;
};

Pool pool_of(const qe_kv_cache_t& c) {
    return {(char*)c.k, (char*)c.v, 2 * c.layer_stride, 2 * c.page_stride, 2 * c.head_stride, 2 * c.token_stride,
            c.layers,   c.pages,    log2_of(c.page),    c.kv_heads,        c.d};
}
Slots slots_of(const qe_kv_cache_t& c) {
    return {c.table, c.length, c.held, c.ref, c.slots, c.width, c.pages, log2_of(c.page)};
}

// sums stop below 2^30, above the number of pages: 1024 entries may ask for more than 2^31
constexpr int kMost = (1 << 30) - 1;
__device__ __forceinline__ int wave_incl_scan(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x = min(x + y, kMost);
    }
    return x;
}
// sum over the threads up to this one, and over all in *total (every thread calls it)
template <int NT>
__device__ int block_incl_scan(int x, int* tmp, int* total) {
    const int incl = wave_incl_scan(x), w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 63) tmp[w] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < NT / 64; i++) {
        if (i < w) before = min(before + tmp[i], kMost);
        all = min(all + tmp[i], kMost);
    }
    *total = all;
    return min(before + incl, kMost);
}

// One block for the whole call: what entry i needs is known from its own slot, where its pages lie in the order of free
// pages from a sum over the entries before it, and the r-th free page from a sum over the threads, each of which counts
// the free pages of a range of its own and puts their numbers into a list, from which a thread gives each one out.
// Latency-bound (dependent reads of seqs, length, table and ref, then the sums): 4 entries of 40 pages 6.3 us, 64 of 16 8.2,
// 1024 of 16 in a pool of 70000 42 (given out by the threads that count them, page after page: 7.0, 14.2 and 138).
__global__ __launch_bounds__(kOne) void reserve_kernel(Slots s, const int32_t* __restrict__ seqs, const int32_t* __restrict__ add,
                                                       int n, int32_t* ok_out, int4* copies) {
    __shared__ __attribute__((aligned(16))) int slot_of[kMaxCacheBatch];
    __shared__ int end_of[kMaxCacheBatch], fresh_of[kMaxCacheBatch], cow_of[kMaxCacheBatch], held_of[kMaxCacheBatch];
    __shared__ int tmp[kOne / 64], list[kList];
    const int i = threadIdx.x, P = 1 << s.shift;
    const int slot = i < n ? seqs[i] : -1;
    const int more = i < n ? add[i] : 0;
    slot_of[i] = slot;
    __syncthreads();
    bool valid = i < n && slot >= 0 && slot < s.slots && more >= 0;
    bool named = false;  // by an earlier entry
    if (valid)
#pragma unroll 4
        for (int j = 0; j < i; j += 4) {
            const int4 o = *reinterpret_cast<const int4*>(slot_of + j);
            named |= (o.x == slot) | ((o.y == slot) & (j + 1 < i)) | ((o.z == slot) & (j + 2 < i)) | ((o.w == slot) & (j + 3 < i));
        }
    valid = valid && !named;
    int need = 0, grow = 0, old = -1, len = 0, held = 0;
    if (valid) {
        len = s.length[slot];
        held = s.held[slot];
        const int64_t want = ((int64_t)len + more + P - 1) >> s.shift;
        valid = len >= 0 && held >= 0 && want <= s.width && held <= s.width;
        if (valid) {
            grow = want > held ? (int)want - held : 0;
            if (more > 0 && (len & (P - 1)) != 0 && (len >> s.shift) < held) {
                const int pg = s.table[(int64_t)slot * s.width + (len >> s.shift)];
                if (pg >= 0 && pg < s.pages && s.ref[pg] > 1) old = pg;
            }
            need = grow + (old >= 0);
        }
    }
    int total, n_free;
    const int end = block_incl_scan<kOne>(need, tmp, &total);
    end_of[i] = end;
    cow_of[i] = old >= 0;
    held_of[i] = held;
    fresh_of[i] = -1;
    // the free pages of this thread's range
    const int per = ((s.pages + kOne - 1) / kOne + 3) & ~3;
    const int p0 = (int)min((int64_t)s.pages, (int64_t)i * per), p1 = (int)min((int64_t)s.pages, (int64_t)p0 + per);
    const bool aligned = ((uintptr_t)s.ref & 15) == 0;
    auto four = [&](int p) {  // pages p .. p + 3 of the range
        int4 r = make_int4(1, 1, 1, 1);
        if (aligned && p + 4 <= p1) {
            r = *reinterpret_cast<const int4*>(s.ref + p);
        } else {
            if (p < p1) r.x = s.ref[p];
            if (p + 1 < p1) r.y = s.ref[p + 1];
            if (p + 2 < p1) r.z = s.ref[p + 2];
            if (p + 3 < p1) r.w = s.ref[p + 3];
        }
        return (uint32_t)((r.x == 0) | (r.y == 0) << 1 | (r.z == 0) << 2 | (r.w == 0) << 3);
    };
    auto free_of = [&](int p) {  // of the 64 pages from p on (of the range): bits of those that are free
        uint64_t bits = 0;
#pragma unroll 4
        for (int k = 0; k < 64 && p + k < p1; k += 4) bits |= (uint64_t)four(p + k) << k;
        return bits;
    };
    int mine = 0;
    uint64_t bits = 0;  // of the range's first 64, all of it in pools of up to 64 K pages
    if (total > 0) {
        bits = free_of(p0);
        mine = __popcll(bits);
        for (int p = p0 + 64; p < p1; p += 64) mine += __popcll(free_of(p));
    }
    int rank = block_incl_scan<kOne>(mine, tmp, &n_free) - mine;
    const bool ok = valid && (need == 0 || end <= n_free);
    // entries are served up to the first that does not fit: the sums only grow
    int given = __syncthreads_or(!ok && need > 0) ? 0 : total;
    if (given == 0 && total > 0) {
        if (i == 0) tmp[0] = 0;
        __syncthreads();
        if (ok && need > 0) atomicMax(&tmp[0], end);
        __syncthreads();
        given = tmp[0];
        __syncthreads();
    }
    // the free pages' numbers in order, kList at a time, then a thread for each of them
    int at = p0;  // where the bits are
    for (int base = 0; base < given; base += kList) {
        const int stop = min(given, base + kList);
        while (rank < stop) {
            if (bits == 0) {
                at += 64;
                if (at >= p1) break;
                bits = free_of(at);
                continue;
            }
            list[rank++ - base] = at + __ffsll((unsigned long long)bits) - 1;
            bits &= bits - 1;
        }
        __syncthreads();
        for (int r = base + i; r < stop; r += kOne) {
            const int p = list[r - base];
            int lo = 0, hi = n - 1;  // the first entry whose pages end behind this one
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (end_of[mid] > r) hi = mid;
                else lo = mid + 1;
            }
            const int nth = r - (lo > 0 ? end_of[lo - 1] : 0);
            if (cow_of[lo] && nth == 0) fresh_of[lo] = p;
            else s.table[(int64_t)slot_of[lo] * s.width + held_of[lo] + nth - cow_of[lo]] = p;
            s.ref[p] = 1;
        }
        __syncthreads();
    }
    const bool copied = ok && old >= 0;
    int n_copies;
    const int c = block_incl_scan<kOne>(copied, tmp, &n_copies) - copied;
    if (copied) {
        s.table[(int64_t)slot * s.width + (len >> s.shift)] = fresh_of[i];
        atomicSub(&s.ref[old], 1);
        copies[1 + c] = make_int4(old, fresh_of[i], len & (P - 1), 0);
    }
    if (ok && grow > 0) s.held[slot] = held + grow;
    if (i < n) ok_out[i] = ok;
    if (i == 0) copies[0] = make_int4(n_copies, 0, 0, 0);
}

// The rows of the pages that reserve copies: a wave per (copy, layer, pool, head), whose rows lie together. As many blocks
// as fill the device go through the list, whose length only the device knows. 96 copies of up to 63 rows in 16 layers: 435 MB
// in 50 us (the parents' rows are read from the caches).
__global__ __launch_bounds__(kThreads) void copy_rows_kernel(Pool p, const int4* __restrict__ copies) {
    const int lane = threadIdx.x & 63, chunks = p.d / 8;  // 16-byte pieces of a row: 8, 16 or 32
    const int64_t per = (int64_t)p.layers * 2 * p.heads, items = per * copies[0].x;
    const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
    for (int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); it < items; it += step) {
        const int4 c = copies[1 + it / per];
        const int r = (int)(it % per), h = r % p.heads, w = r / p.heads;
        const int64_t off = (int64_t)(w >> 1) * p.layer + (int64_t)h * p.head;
        char* base = (w & 1 ? p.v : p.k) + off;
        const char* src = base + (int64_t)c.x * p.page;
        char* dst = base + (int64_t)c.y * p.page;
        const int pieces = c.z * chunks;
        for (int i = lane; i < pieces; i += 256) {
            u32x4_v x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int q = i + 64 * u;
                if (q < pieces) x[u] = *reinterpret_cast<const u32x4_v*>(src + (int64_t)(q / chunks) * p.token + q % chunks * 16);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int q = i + 64 * u;
                if (q < pieces) *reinterpret_cast<u32x4_v*>(dst + (int64_t)(q / chunks) * p.token + q % chunks * 16) = x[u];
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void fork_kernel(Slots s, const int32_t* __restrict__ parents,
                                                        const int32_t* __restrict__ children, int n, int32_t* ok_out) {
    const int i = blockIdx.x, par = parents[i], kid = children[i];
    bool bad = par < 0 || par >= s.slots || kid < 0 || kid >= s.slots;
    for (int j = threadIdx.x; j < n; j += kThreads) bad = bad || (j < i && children[j] == kid) || children[j] == par;
    int len = 0, keep = 0;
    if (!bad) {
        len = s.length[par];
        keep = (int)(((int64_t)len + (1 << s.shift) - 1) >> s.shift);
        bad = len < 0 || keep > s.held[par] || keep > s.width || s.held[kid] != 0 || s.length[kid] != 0;
    }
    if (__syncthreads_or(bad)) {  // also: every thread has read what thread 0 writes below
        if (threadIdx.x == 0) ok_out[i] = 0;
        return;
    }
    for (int j = threadIdx.x; j < keep; j += kThreads) {
        const int pg = s.table[(int64_t)par * s.width + j];
        s.table[(int64_t)kid * s.width + j] = pg;
        if (pg >= 0 && pg < s.pages) atomicAdd(&s.ref[pg], 1);
    }
    if (threadIdx.x == 0) {
        s.length[kid] = len;
        s.held[kid] = keep;
        ok_out[i] = 1;
    }
}

__global__ __launch_bounds__(kThreads) void release_kernel(Slots s, const int32_t* __restrict__ seqs,
                                                           const int32_t* __restrict__ lengths) {
    const int i = blockIdx.x, slot = seqs[i];
    bool skip = slot < 0 || slot >= s.slots;
    for (int j = threadIdx.x; j < i; j += kThreads) skip = skip || seqs[j] == slot;
    int len = 0, held = 0;
    if (!skip) {
        len = min(max(s.length[slot], 0), lengths ? max(lengths[i], 0) : 0);
        held = min(max(s.held[slot], 0), s.width);
    }
    if (__syncthreads_or(skip)) return;
    const int keep = min(held, (int)(((int64_t)len + (1 << s.shift) - 1) >> s.shift));
    for (int j = keep + threadIdx.x; j < held; j += kThreads) {
        int32_t* t = s.table + (int64_t)slot * s.width + j;
        const int pg = *t;
        *t = -1;
        if (pg >= 0 && pg < s.pages) atomicSub(&s.ref[pg], 1);
    }
    if (threadIdx.x == 0) {
        s.length[slot] = len;
        s.held[slot] = keep;
    }
}

struct AppendArgs {
    const char *k, *v;
    int64_t kl, kr, kh, vl, vr, vh;  // bytes
    int layer0, nseq, first, t;  // rows first .. t - 1
};
// A wave per row and layer: its lanes find the row's sequence with one vote per 64 sequences, then move the row's keys and
// values, 16 bytes a lane. 2048 rows, 32 layers, 8 heads of 128: 537 MB in 101-105 us.
__global__ __launch_bounds__(kThreads) void append_kernel(Pool p, Slots s, AppendArgs a, const int32_t* __restrict__ seqs,
                                                          const int32_t* __restrict__ cu) {
    const int lane = threadIdx.x & 63;
    const int t = a.first + blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (t >= a.t) return;
    int b = 0;
    for (int j = 0; j < a.nseq; j += 64) b += __popcll(__ballot(j + lane < a.nseq && cu[j + lane + 1] <= t));
    if (b >= a.nseq || t < cu[b]) return;
    const int slot = seqs[b];
    if (slot < 0 || slot >= s.slots) return;
    const int64_t pos = (int64_t)s.length[slot] + t - cu[b], idx = pos >> s.shift;
    if (pos < 0 || idx >= s.held[slot] || idx >= s.width) return;
    const int pg = s.table[(int64_t)slot * s.width + idx];
    if (pg < 0 || pg >= p.pages || s.ref[pg] > 1) return;  // never into a page that other slots hold too
    const int chunks = p.d / 8, each = p.heads * chunks;
    const int64_t to = (int64_t)(a.layer0 + blockIdx.y) * p.layer + (int64_t)pg * p.page + (pos & ((1 << s.shift) - 1)) * p.token;
    const char* ks = a.k + blockIdx.y * a.kl + t * a.kr;
    const char* vs = a.v + blockIdx.y * a.vl + t * a.vr;
    for (int i = lane; i < each; i += 64) {
        const int h = i / chunks, o = i % chunks * 16;
        const u32x4_v x = *reinterpret_cast<const u32x4_v*>(ks + h * a.kh + o);
        const u32x4_v y = *reinterpret_cast<const u32x4_v*>(vs + h * a.vh + o);
        *reinterpret_cast<u32x4_v*>(p.k + to + h * p.head + o) = x;
        *reinterpret_cast<u32x4_v*>(p.v + to + h * p.head + o) = y;
    }
}

// A wave per (sequence, layer, pool, head) holds all of its path's rows in registers before it writes the first, so the
// path may have any order.
template <int D>
__global__ __launch_bounds__(kThreads) void accept_rows_kernel(Pool p, Slots s, const int32_t* __restrict__ seqs,
                                                               const int32_t* __restrict__ count,
                                                               const int32_t* __restrict__ path, int most) {
    constexpr int CH = D / 8, ROWS = 64 / CH, MAXI = kMaxTreeNodes / ROWS;
    const int lane = threadIdx.x & 63, i = blockIdx.z;
    const int w = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);  // pool and head
    if (w >= 2 * p.heads) return;
    const int slot = seqs[i];
    if (slot < 0 || slot >= s.slots) return;
    const int len = s.length[slot], held = min(s.held[slot], s.width), n = min(count[i], most);
    // lane j: where row path[j] lies and where it goes, -1: nothing to move
    int64_t from = -1, to = -1;
    if (lane < n && len >= 0) {
        const int j = path[(int64_t)i * most + lane];
        const int64_t a = (int64_t)len + j, b = (int64_t)len + lane;
        if (j >= 0 && j != lane && (a >> s.shift) < held && (b >> s.shift) < held) {
            const int pa = s.table[(int64_t)slot * s.width + (a >> s.shift)], pb = s.table[(int64_t)slot * s.width + (b >> s.shift)];
            if (pa >= 0 && pa < p.pages && pb >= 0 && pb < p.pages && s.ref[pb] <= 1) {
                from = pa * p.page + (a & ((1 << s.shift) - 1)) * p.token;
                to = pb * p.page + (b & ((1 << s.shift) - 1)) * p.token;
            }
        }
    }
    char* base = (w & 1 ? p.v : p.k) + (int64_t)blockIdx.y * p.layer + (int64_t)(w >> 1) * p.head + lane % CH * 16;
    u32x4_v x[MAXI];
#pragma unroll
    for (int u = 0; u < MAXI; u++) {
        if (u * ROWS >= n) continue;
        const int64_t f = __shfl(from, u * ROWS + lane / CH);
        if (f >= 0) x[u] = *reinterpret_cast<const u32x4_v*>(base + f);
    }
    // every row is in registers before the first store of the wave: a row's place may be another row's source
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < MAXI; u++) {
        if (u * ROWS >= n) continue;
        const int64_t d = __shfl(to, u * ROWS + lane / CH);
        if (d >= 0) *reinterpret_cast<u32x4_v*>(base + d) = x[u];
    }
}

__global__ __launch_bounds__(kThreads) void accept_length_kernel(Slots s, const int32_t* __restrict__ seqs,
                                                                 const int32_t* __restrict__ count, int most, int n, int32_t* out) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const int slot = seqs[i];
    if (slot < 0 || slot >= s.slots) return;
    const int64_t room = (int64_t)min(max(s.held[slot], 0), s.width) << s.shift;
    const int64_t len = s.length[slot], c = max(count[i], 0);
    out[slot] = (int)max(len, min(len + (most >= 0 ? min(c, (int64_t)most) : c), room));
}
}  // namespace

void kv_check(const qe_kv_cache_t* c, const char* who) {
    CHECK(c != nullptr, "%s: no cache", who);
    CHECK(c->k && c->v && c->table && c->length && c->held && c->ref, "%s: null pointer in the cache", who);
    CHECK((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "%s: pools must be 16-byte aligned", who);
    CHECK(c->layers >= 1 && c->pages >= 1 && c->slots >= 1 && c->width >= 1 && c->kv_heads >= 1 && c->kv_heads <= 1024,
          "%s: cache of layers %d pages %d slots %d width %d kv_heads %d", who, c->layers, c->pages, c->slots, c->width, c->kv_heads);
    CHECK(c->d == 64 || c->d == 128 || c->d == 256, "%s: d %d (64, 128 or 256)", who, c->d);
    CHECK(c->page >= 16 && c->page <= 1024 && (c->page & (c->page - 1)) == 0, "%s: page %d (a power of two, 16 .. 1024)", who, c->page);
    CHECK(c->layer_stride % 8 == 0 && c->page_stride % 8 == 0 && c->head_stride % 8 == 0 && c->token_stride % 8 == 0,
          "%s: cache strides must be multiples of 8", who);
    CHECK((int64_t)c->width * c->page <= (int64_t)1 << 30, "%s: width %d pages of %d pass 2^30 tokens", who, c->width, c->page);
    CHECK(c->pages < 1 << 29, "%s: %d pages (below 2^29)", who, c->pages);
    CHECK(c->token_stride >= 0 && c->token_stride < 1 << 24, "%s: tokens %lld elements apart (below 2^24)", who, (long long)c->token_stride);
    CHECK(c->f16 == 0 || c->f16 == 1, "%s: f16 %d", who, c->f16);
}

static void check_batch(const char* who, int n) { CHECK(n >= 0 && n <= kMaxCacheBatch, "%s: n = %d (at most %d)", who, n, kMaxCacheBatch); }

void kv_reserve(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* add, int n, int32_t* ok, int32_t* copies,
                hipStream_t st) {
    check_batch("qe_kv_reserve", n);
    CHECK(copies && ((uintptr_t)copies & 15) == 0 && (n == 0 || (seqs && add && ok)), "qe_kv_reserve: null or unaligned pointer");
    if (n == 0) return;
    reserve_kernel<<<1, kOne, 0, st>>>(slots_of(c), seqs, add, n, ok, reinterpret_cast<int4*>(copies));
    HIP_CHECK(hipGetLastError());
    const int64_t waves = (int64_t)n * c.layers * 2 * c.kv_heads;
    const int grid = (int)std::min<int64_t>((waves + 3) / 4, 8 * qe_num_cus());
    copy_rows_kernel<<<grid, kThreads, 0, st>>>(pool_of(c), reinterpret_cast<const int4*>(copies));
    HIP_CHECK(hipGetLastError());
}

void kv_fork(const qe_kv_cache_t& c, const int32_t* parents, const int32_t* children, int n, int32_t* ok, hipStream_t st) {
    check_batch("qe_kv_fork", n);
    CHECK(n == 0 || (parents && children && ok), "qe_kv_fork: null pointer");
    if (n == 0) return;
    fork_kernel<<<n, kThreads, 0, st>>>(slots_of(c), parents, children, n, ok);
    HIP_CHECK(hipGetLastError());
}

void kv_release(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* lengths, int n, hipStream_t st) {
    check_batch("qe_kv_release", n);
    CHECK(n == 0 || seqs, "qe_kv_release: null pointer");
    if (n == 0) return;
    release_kernel<<<n, kThreads, 0, st>>>(slots_of(c), seqs, lengths);
    HIP_CHECK(hipGetLastError());
}

void kv_append(const qe_kv_cache_t& c, int layer, int layers, const void* k, const void* v, const int64_t* strides,
               const int32_t* seqs, const int32_t* cu, int nseq, int t, hipStream_t st) {
    CHECK(layer >= 0 && layers >= 1 && layer <= c.layers - layers, "qe_kv_append: layers %d .. %d of %d", layer, layer + layers, c.layers);
    CHECK(nseq >= 0 && t >= 0 && t <= kMaxRows && layers <= 65535, "qe_kv_append: nseq %d t %d layers %d", nseq, t, layers);
    if (nseq == 0 || t == 0) return;
    CHECK(k && v && strides && seqs && cu, "qe_kv_append: null pointer");
    CHECK((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "qe_kv_append: k and v must be 16-byte aligned");
    for (int i = 0; i < 6; i++) CHECK(strides[i] % 8 == 0, "qe_kv_append: stride %lld (a multiple of 8)", (long long)strides[i]);
    AppendArgs a{(const char*)k, (const char*)v, 2 * strides[0], 2 * strides[1], 2 * strides[2], 2 * strides[3], 2 * strides[4],
                 2 * strides[5], layer, nseq, 0, 0};
    constexpr int kLaunch = 1 << 25;  // rows of a launch: a grid has fewer than 2^32 threads in x, 64 a row
    for (int first = 0; first < t; first += kLaunch) {
        a.first = first;
        a.t = std::min(t, first + kLaunch);
        append_kernel<<<dim3((a.t - first - 1) / (kThreads / 64) + 1, layers), kThreads, 0, st>>>(pool_of(c), slots_of(c), a, seqs, cu);
        HIP_CHECK(hipGetLastError());
    }
}

void kv_accept(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* count, const int32_t* path, int most, int n,
               int32_t* length, hipStream_t st) {
    CHECK(n >= 0 && n <= 65535, "qe_kv_accept: n = %d", n);
    CHECK(c.layers <= 65535, "qe_kv_accept: %d layers", c.layers);
    if (n == 0) return;
    CHECK(seqs && count, "qe_kv_accept: null pointer");
    if (path) {
        CHECK(most >= 0 && most <= kMaxTreeNodes, "qe_kv_accept: paths of %d (at most %d)", most, kMaxTreeNodes);
        if (most > 0) {
            const Pool p = pool_of(c);
            const Slots s = slots_of(c);
            const dim3 grid((2 * c.kv_heads + 3) / 4, c.layers, n);
            if (c.d == 64) accept_rows_kernel<64><<<grid, kThreads, 0, st>>>(p, s, seqs, count, path, most);
            else if (c.d == 128) accept_rows_kernel<128><<<grid, kThreads, 0, st>>>(p, s, seqs, count, path, most);
            else accept_rows_kernel<256><<<grid, kThreads, 0, st>>>(p, s, seqs, count, path, most);
            HIP_CHECK(hipGetLastError());
        }
    }
    accept_length_kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, st>>>(slots_of(c), seqs, count, path ? most : -1, n,
                                                                              length ? length : c.length);
    HIP_CHECK(hipGetLastError());
}
