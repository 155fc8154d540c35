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
    // whether all of the queries see the whole page
    __device__ __forceinline__ bool all_see(int pg) const {
        const int first = pg * PR_PAGE, last = first + PR_PAGE - 1;
        return last <= pos_lo && last < key_end && (pos_hi - first < window || last < sinks);
    }
    // whether any of the queries sees the key: the last one sees the newest keys,
    // the first one's window reaches back furthest
    __device__ __forceinline__ bool any_sees(int key) const {
        return key <= pos_hi && key < key_end && (pos_lo - key < window || key < sinks);
    }
};

// skip: pages before this one are somebody else's business (sinks then 0)
__device__ __forceinline__ PageList page_list(int pos_lo, int pos_hi, int window, int sinks,
                                              int bt_width, int skip = 0) {
    PageList l;
    l.pos_lo = pos_lo; l.pos_hi = pos_hi; l.window = window; l.sinks = sinks;
    l.key_end = bt_width * PR_PAGE;
    const int end_key = min(pos_hi + 1, l.key_end);          // keys [0, end_key)
    const int n_pages = end_key <= 0 ? 0 : (end_key + PR_PAGE - 1) / PR_PAGE;
    l.n_first = min((min(sinks, l.key_end) + PR_PAGE - 1) / PR_PAGE, n_pages);
    // first key in the first query's window, rounded down to its page
    const int lo_key = window > pos_lo ? 0 : pos_lo - window + 1;
    const int from = max(max(lo_key / PR_PAGE, l.n_first), skip);
    // window 0: nobody's window holds a key
    const int recent = window > 0 ? max(n_pages - from, 0) : 0;
    l.shift = from - l.n_first;
    l.n = l.n_first + recent;
    return l;
}

// Row `at` of several partial results: channels d .. d + 3 of O, with the maximum (in
// log2 units) and the sum.  A part that saw nothing carries l = 0 and no O; a sum of NaN
// makes the row NaN.
struct PartSum {
    float m, l;
    float4 o;
};
__device__ __forceinline__ PartSum join_parts(const float* o, const float* ml, int64_t rows,
                                              int parts, int64_t at, int d) {
    PartSum r = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    // eight parts' loads in flight at a time, none waiting for another
    for (int s0 = 0; s0 < parts; s0 += 8) {
        float2 x[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = (int64_t)min(s0 + k, parts - 1) * rows + at;
            x[k] = *reinterpret_cast<const float2*>(ml + 2 * i);
            v[k] = *reinterpret_cast<const float4*>(o + i * PR_HD + d);
        }
        float up = r.m;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (s0 + k >= parts) x[k].y = 0.f;
            if (x[k].y != 0.f) up = fmaxf(up, x[k].x);
        }
        const float a = r.l != 0.f ? pr_exp2(r.m - up) : 0.f;
        r.l *= a;
        r.o.x *= a; r.o.y *= a; r.o.z *= a; r.o.w *= a;
        r.m = up;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (x[k].y != 0.f) {                // (a part without keys wrote no O)
                const float w = pr_exp2(x[k].x - up);
                r.l += w * x[k].y;
                r.o.x += w * v[k].x; r.o.y += w * v[k].y;
                r.o.z += w * v[k].z; r.o.w += w * v[k].w;
            }
        }
    }
    return r;
}
#endif

struct RowAttnParams {
    const __nv_bfloat16* q;
    int64_t q_tok, q_head;
    const __nv_bfloat16 *k, *v;
    int64_t sb, st, sh;               // cache strides: block, token, KV head
    const int32_t* table;
    int64_t bt_stride;
    int bt_width, num_blocks, n_tok;  // n_tok: rows of q and out
    const int32_t* cu_q;              // null: request r's one token is row r
    const int32_t* seq_lens;
    __nv_bfloat16* out;
    int64_t o_tok, o_head;
    float* lse;                       // optional, lse[token * lse_tok + head]
    int64_t lse_tok;
    int n_kv, G, window, sinks;
    float scale_log2;                 // softmax scale * log2(e)
    int max_rows;                     // requests with more rows (tokens x G) are left out
    int beside;                       // the launch before this one is the call's tiled kernel
    // shared prefix: (n_groups + 1) row bounds, or null; the whole pages of the prefix are
    // left out, and the result becomes part number `part` (layout: TileAttnParams)
    const int32_t* cu_groups;
    const int32_t* prefix_lens;
    int n_groups, part;
    int64_t part_rows;
    float *parts_o, *parts_ml;
};

// the tiled kernel: segments bounds[s] .. bounds[s + 1] of query tokens
struct TileAttnParams {
    RowAttnParams r;
    const int32_t* bounds;            // cu_q, or cu_groups of a shared prefix
    const int32_t* prefix_lens;       // shared prefix: tokens of the segment's prefix
    int n_seg, min_rows;              // windowed: segments of up to min_rows rows are left out
    // key tiles cut into `parts`: O relative to its maximum (parts, part_rows, 128) and
    // (maximum in log2 units, sum) pairs (parts, part_rows, 2); null: one part, final
    int parts;
    int64_t part_rows;
    float *parts_out, *parts_ml;
    int* status;
    int head_chunks;                  // 64-channel chunks between two heads
    int tile_bound, tile_more;        // row tiles expected and possible beyond; 0: count them
};

// csrc/row_attn.cu; `who` names the entry point in error messages, most_rows: about how
// many rows the longest request has that the launch serves (any number is served).
// splits > 1: that many CTAs to a pair, whose results become parts p.part ..
int launch_row_attn(const char* who, const RowAttnParams& p, int n_req, int most_rows,
                    int splits, cudaStream_t s);
// csrc/tile_attn.cu; tiles: row tiles expected, max_tiles: there are no more than this
int launch_tile_attn(const char* who, TileAttnParams p, int tiles, int max_tiles, int n_tok,
                     cudaStream_t s);
int launch_join_parts(const char* who, const TileAttnParams& p, int parts, int n_tok,
                      cudaStream_t s);

}  // namespace locks
