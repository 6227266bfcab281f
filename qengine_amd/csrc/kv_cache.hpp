// The paged cache of keys and values on the device (qe_kv_cache_t of include/qe_kernels.h) as the kernels take it.
#pragma once
#include "../../include/qe_kernels.h"
#include "qe_api.hpp"

constexpr int kMaxCacheBatch = 1024;  // sequences of one reserve, fork or release call (one block looks at all of them)
constexpr int kMaxRows = 1 << 30;     // rows of one append or attention call: row numbers and their tiles' ends fit 32 bits
constexpr int kMaxTreeNodes = 64;     // drafted tokens of a sequence: the bits of a mask word
constexpr int kMaxTreeBatch = 4096;   // sequences of one attention call (their tile counts are summed in LDS)

// aborts with a message on a description that no kernel can run on
void kv_check(const qe_kv_cache_t* c, const char* who);

inline int log2_of(int p) {
    int s = 0;
    while ((1 << s) < p) s++;
    return s;
}

void kv_reserve(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* add, int n, int32_t* ok, int32_t* copies,
                hipStream_t st);
void kv_fork(const qe_kv_cache_t& c, const int32_t* parents, const int32_t* children, int n, int32_t* ok, hipStream_t st);
void kv_release(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* lengths, int n, hipStream_t st);
void kv_append(const qe_kv_cache_t& c, int layer, int layers, const void* k, const void* v, const int64_t* strides,
               const int32_t* seqs, const int32_t* cu, int nseq, int t, hipStream_t st);
void kv_accept(const qe_kv_cache_t& c, const int32_t* seqs, const int32_t* count, const int32_t* path, int most, int n,
               int32_t* length, hipStream_t st);

struct AttnPromptArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // strides in elements
    const int32_t* cu;
    int nseq, t, heads, kv_heads, d;
    float scale;
};
void attn_prompt(const AttnPromptArgs& a, bool f16, hipStream_t st);

struct AttnTreeArgs {
    const void* q;
    void* out;
    float* lse;
    int64_t q_row, q_head, o_row, o_head;
    const int32_t *seqs, *cu;
    int nseq, t, max_new;
    const uint64_t* mask;
    int heads;
    float scale;
};
void attn_tree(const qe_kv_cache_t& c, int layer, const AttnTreeArgs& a, hipStream_t st);
// off: as where the device has no memory for the parts of rows (a test hook)
void attn_tree_set_split(bool on);
bool attn_tree_split();
