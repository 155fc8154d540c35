// What the windowed and the shared-prefix attention kernels have in common: which
// keys a query sees, the list of pages a block of queries has to read, and the
// arguments of the few-row kernel.
#pragma once
#include "common.cuh"

namespace locks {

constexpr int PR_HD = 128;
constexpr int PR_PAGE = 16;
constexpr float PR_LOG2E = 1.4426950408889634f;
constexpr float PR_LN2 = 0.6931471805599453f;

#ifdef __CUDACC__
__device__ __forceinline__ float pr_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The pages that queries at positions [lo, hi] can see: the first pages (up to
// `n_first` of them) and the recent ones, walked as one list of n entries.
struct PageList {
    int n, n_first, shift;        // entry v is page v, or v + shift from n_first on
    int pos_lo, pos_hi, window, sinks, key_end;

    __device__ __forceinline__ int page(int v) const {
        return v < n_first ? v : v + shift;
    }
    __device__ __forceinline__ bool sees(int key, int pos) const {
        // (pos - key < window: no overflow for key >= 0, pos < 2^31)
        return key <= pos && key < key_end && (pos - key < window || key < sinks);
    }
    // whether any of the queries sees the key: the last one sees the newest keys,
    // the first one's window reaches back furthest
    __device__ __forceinline__ bool any_sees(int key) const {
        return key <= pos_hi && key < key_end && (pos_lo - key < window || key < sinks);
    }
};

__device__ __forceinline__ PageList page_list(int pos_lo, int pos_hi, int window, int sinks,
                                              int bt_width) {
    PageList l;
    l.pos_lo = pos_lo; l.pos_hi = pos_hi; l.window = window; l.sinks = sinks;
    l.key_end = bt_width * PR_PAGE;
    const int end_key = min(pos_hi + 1, l.key_end);          // keys [0, end_key)
    const int n_pages = end_key <= 0 ? 0 : (end_key + PR_PAGE - 1) / PR_PAGE;
    l.n_first = min((min(sinks, l.key_end) + PR_PAGE - 1) / PR_PAGE, n_pages);
    // first key in the first query's window, rounded down to its page
    const int lo_key = window > pos_lo ? 0 : pos_lo - window + 1;
    const int from = max(lo_key / PR_PAGE, l.n_first);
    // window 0: nobody's window holds a key
    const int recent = window > 0 ? max(n_pages - from, 0) : 0;
    l.shift = from - l.n_first;
    l.n = l.n_first + recent;
    return l;
}
#endif

struct RowAttnParams {
    const __nv_bfloat16* q;
    int64_t q_tok, q_head;
    const __nv_bfloat16 *k, *v;
    int64_t sb, st, sh;               // cache strides: block, token, KV head
    const int32_t* table;
    int64_t bt_stride;
    int bt_width, num_blocks;
    const int32_t* cu_q;              // null: request r's one token is row r
    const int32_t* seq_lens;
    __nv_bfloat16* out;
    int64_t o_tok, o_head;
    float* lse;                       // optional, lse[token * lse_tok + head]
    int64_t lse_tok;
    int n_kv, G, window, sinks;
    float scale_log2;                 // softmax scale * log2(e)
    const int32_t* cu_groups;         // shared prefix: (n_groups + 1) row bounds, or null
    int n_groups;
};

// csrc/row_attn.cu; `who` names the entry point in error messages
int launch_row_attn(const char* who, const RowAttnParams& p, int n_req, cudaStream_t s);

}  // namespace locks
