// Entry points of the windowed and the shared-prefix attention over the paged cache.
#include "common.cuh"
#include "paged_rows.cuh"

namespace locks {
namespace {

bool rows16(const void* p, int64_t a, int64_t b) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a % 8 == 0 && b % 8 == 0;
}

// the checks both entry points share
int check_paged(const char* who, const RowAttnParams& p, int n_req, int head_dim, int page,
                const float* scratch, int64_t scratch_floats) {
    LOCKS_REQUIRE(p.q && p.k && p.v && p.table && p.seq_lens && p.out, LOCKS_ERR_ARG,
                  "%s: null pointer argument", who);
    LOCKS_REQUIRE(head_dim == PR_HD && page == PR_PAGE, LOCKS_ERR_GEOMETRY,
                  "%s: supports head_dim 128 / page 16, got %d / %d", who, head_dim, page);
    LOCKS_REQUIRE(p.G >= 1 && p.G <= 16, LOCKS_ERR_GEOMETRY,
                  "%s: supports 1 <= G <= 16, got %d", who, p.G);
    LOCKS_REQUIRE(n_req >= 0 && n_req <= 65535 && p.n_kv >= 1 && p.n_kv <= 65535 &&
                      p.bt_width >= 1 && p.bt_width <= (1 << 26) && p.num_blocks >= 1 &&
                      p.sinks >= 0 && p.window >= 0 && scratch_floats >= 0,
                  LOCKS_ERR_ARG, "%s: bad size argument", who);
    LOCKS_REQUIRE(rows16(p.q, p.q_tok, p.q_head) && rows16(p.k, p.st, p.sh) &&
                      rows16(p.v, p.sb, 0) && rows16(p.out, p.o_tok, p.o_head),
                  LOCKS_ERR_ARG, "%s: rows must be 16-byte aligned", who);
    LOCKS_REQUIRE(p.n_kv == 1 || (p.sh % 64 == 0 && p.sh > 0 && p.sh < ((int64_t)1 << 30)),
                  LOCKS_ERR_GEOMETRY, "%s: the head stride must be a multiple of 64", who);
    LOCKS_REQUIRE(p.st > 0 && p.sb > 0, LOCKS_ERR_ARG, "%s: bad cache stride", who);
    LOCKS_REQUIRE((reinterpret_cast<uintptr_t>(scratch) & 15) == 0, LOCKS_ERR_ARG,
                  "%s: scratch must be 16-byte aligned", who);
    return LOCKS_OK;
}

// Requests of up to this many rows (query tokens x G) go to the few-row kernel, whose
// fragments hold 16; above it the tiled kernel takes 128 rows at a time.
constexpr int FEW_ROWS = 16;
constexpr int TILE_ROWS = 256, TILE_PAGES = 8;
// Few (request, KV head) pairs whose lists may be this long are worth more CTAs than a
// cluster has, and a launch that joins their parts (3 us).  8 pairs, in clusters and in
// parts: 2048 pages 36 and 32 us, 4096 pages 64 and 53, 8192 pages 122 and 96; 2 pairs x
// 8192 pages 87 and 46.
constexpr int LONG_PAGES = 2048;

// How many parts the key tiles are cut into: enough CTAs for the device, at least two
// tiles a part (one per stream), as many as the scratch has room for.
int parts_for(int64_t ctas, int64_t key_pages, int64_t part_floats, int64_t scratch_floats) {
    const int64_t tiles = (key_pages + TILE_PAGES - 1) / TILE_PAGES;
    int64_t n = sm_count() / (ctas > 0 ? ctas : 1);
    n = n < tiles / 2 ? n : tiles / 2;
    const int64_t room = scratch_floats / part_floats;
    n = n < room ? n : room;
    return n < 1 ? 1 : (int)n;
}

}  // namespace
}  // namespace locks

using namespace locks;

extern "C" int locks_window_attention(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
    const void* v_cache, int64_t kv_stride_block, int64_t kv_stride_tok,
    int64_t kv_stride_head, const int32_t* block_table, int64_t bt_stride, int bt_width,
    int num_blocks, const int32_t* cu_q, const int32_t* seq_lens, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, float* lse, int64_t lse_stride_tok,
    float* scratch, int64_t scratch_floats, int n_tok, int n_req, int max_q, int n_kv,
    int G, int head_dim, int page, int window, int sinks, float scale, int* status,
    locks_stream_t stream) {
    RowAttnParams p = {};
    p.q = static_cast<const __nv_bfloat16*>(q); p.q_tok = q_stride_tok; p.q_head = q_stride_head;
    p.k = static_cast<const __nv_bfloat16*>(k_cache);
    p.v = static_cast<const __nv_bfloat16*>(v_cache);
    p.sb = kv_stride_block; p.st = kv_stride_tok; p.sh = kv_stride_head;
    p.table = block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
    p.num_blocks = num_blocks; p.n_tok = n_tok; p.cu_q = cu_q; p.seq_lens = seq_lens;
    p.out = static_cast<__nv_bfloat16*>(out); p.o_tok = o_stride_tok; p.o_head = o_stride_head;
    p.lse = lse; p.lse_tok = lse_stride_tok;
    p.n_kv = n_kv; p.G = G; p.window = window; p.sinks = sinks;
    p.scale_log2 = scale * PR_LOG2E;
    const char* who = "locks_window_attention";
    const int rc = check_paged(who, p, n_req, head_dim, page, scratch, scratch_floats);
    if (rc != LOCKS_OK) return rc;
    LOCKS_REQUIRE(cu_q, LOCKS_ERR_ARG, "%s: null pointer argument", who);
    LOCKS_REQUIRE(n_tok >= 0 && max_q >= 0, LOCKS_ERR_ARG, "%s: bad size argument", who);
    LOCKS_REQUIRE(scale > 0.f, LOCKS_ERR_ARG, "%s: scale must be positive", who);
    if (n_req == 0 || n_tok == 0 || max_q == 0) return LOCKS_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.max_rows = INT32_MAX;
    const int64_t span = (int64_t)window + sinks + max_q;
    const int64_t pages = span / page + 2 < bt_width ? span / page + 2 : bt_width;
    TileAttnParams tp = {};
    tp.part_rows = (int64_t)n_tok * n_kv * G;
    if ((int64_t)max_q * G > FEW_ROWS) {
        // (how the tokens fall on the requests is known on the device only: an upper
        // bound of the tiles, CTAs without one return at once.  max_q may be too small:
        // it lowers the count that is expected, not the bound)
        const int64_t rows = (int64_t)n_tok * G;
        const int64_t many = rows / (FEW_ROWS + 1) < n_req ? rows / (FEW_ROWS + 1) : n_req;
        const int64_t bound = (rows + (TILE_ROWS - 1) * many) / TILE_ROWS;
        const int64_t most = many * (((int64_t)max_q * G + TILE_ROWS - 1) / TILE_ROWS);
        const int64_t tiles = bound < most ? bound : most;
        if (bound > 0) {
            p.max_rows = FEW_ROWS;
            tp.r = p;
            tp.bounds = cu_q; tp.n_seg = n_req; tp.min_rows = FEW_ROWS; tp.status = status;
            tp.parts = scratch ? parts_for(tiles * n_kv, pages, tp.part_rows * (PR_HD + 2),
                                           scratch_floats) : 1;
            if (tp.parts > 1) {
                tp.parts_out = scratch;
                tp.parts_ml = scratch + tp.parts * tp.part_rows * PR_HD;
            }
            p.beside = 1;
            int rc2 = launch_tile_attn(who, tp, (int)tiles, (int)bound, n_tok, s);
            if (rc2 == LOCKS_OK)
                rc2 = launch_row_attn(who, p, n_req, max_q < FEW_ROWS ? max_q * G : FEW_ROWS, 1,
                                      s);
            if (rc2 == LOCKS_OK && tp.parts > 1) rc2 = launch_join_parts(who, tp, tp.parts, n_tok, s);
            return rc2;
        }
    }
    const int64_t pairs = (int64_t)n_req * n_kv;
    int64_t splits = scratch ? scratch_floats / (tp.part_rows * (PR_HD + 2)) : 0;
    splits = splits < 2 * sm_count() / pairs ? splits : 2 * sm_count() / pairs;
    if (pages < LONG_PAGES || splits < 4)
        return launch_row_attn(who, p, n_req, max_q < FEW_ROWS ? max_q * G : FEW_ROWS, 1, s);
    p.part_rows = tp.part_rows;
    p.parts_o = scratch;
    p.parts_ml = scratch + splits * tp.part_rows * PR_HD;
    tp.r = p;
    tp.bounds = cu_q; tp.n_seg = n_req; tp.min_rows = -1;       // (no tiles: all rows joined)
    tp.parts_out = p.parts_o; tp.parts_ml = p.parts_ml;
    const int rc2 = launch_row_attn(
        who, p, n_req, max_q < FEW_ROWS ? max_q * G : FEW_ROWS, (int)splits, s);
    return rc2 == LOCKS_OK ? launch_join_parts(who, tp, (int)splits, n_tok, s) : rc2;
}

extern "C" int locks_shared_prefix_decode(
    const void* q, int64_t q_stride_req, int64_t q_stride_head, const void* k_cache,
    const void* v_cache, int64_t kv_stride_block, int64_t kv_stride_tok,
    int64_t kv_stride_head, const int32_t* block_table, int64_t bt_stride, int bt_width,
    int num_blocks, const int32_t* seq_lens, const int32_t* cu_groups,
    const int32_t* prefix_lens, void* out, int64_t o_stride_req, int64_t o_stride_head,
    float* lse, int64_t lse_stride_req, float* scratch, int64_t scratch_floats, int n_req,
    int n_groups, int n_kv, int G, int head_dim, int page, float scale, int* status,
    locks_stream_t stream) {
    RowAttnParams p = {};
    p.q = static_cast<const __nv_bfloat16*>(q); p.q_tok = q_stride_req; p.q_head = q_stride_head;
    p.k = static_cast<const __nv_bfloat16*>(k_cache);
    p.v = static_cast<const __nv_bfloat16*>(v_cache);
    p.sb = kv_stride_block; p.st = kv_stride_tok; p.sh = kv_stride_head;
    p.table = block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
    p.num_blocks = num_blocks; p.n_tok = n_req; p.seq_lens = seq_lens;
    p.out = static_cast<__nv_bfloat16*>(out); p.o_tok = o_stride_req; p.o_head = o_stride_head;
    p.lse = lse; p.lse_tok = lse_stride_req;
    p.n_kv = n_kv; p.G = G; p.window = INT32_MAX; p.sinks = 0;
    p.scale_log2 = scale * PR_LOG2E;
    p.cu_groups = cu_groups; p.n_groups = n_groups; p.prefix_lens = prefix_lens;
    const char* who = "locks_shared_prefix_decode";
    const int rc = check_paged(who, p, n_req, head_dim, page, scratch, scratch_floats);
    if (rc != LOCKS_OK) return rc;
    LOCKS_REQUIRE(cu_groups && prefix_lens && scratch, LOCKS_ERR_ARG,
                  "%s: null pointer argument", who);
    LOCKS_REQUIRE(n_groups >= 0, LOCKS_ERR_ARG, "%s: bad size argument", who);
    LOCKS_REQUIRE(scratch_floats >= (int64_t)n_req * n_kv * G * (PR_HD + 2) * 2, LOCKS_ERR_SIZE,
                  "%s: scratch holds %lld floats, at least %lld are needed", who,
                  (long long)scratch_floats, (long long)n_req * n_kv * G * (PR_HD + 2) * 2);
    LOCKS_REQUIRE(scale > 0.f, LOCKS_ERR_ARG, "%s: scale must be positive", who);
    if (n_req == 0 || n_groups == 0) return LOCKS_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    TileAttnParams tp = {};
    tp.r = p;
    tp.bounds = cu_groups; tp.prefix_lens = prefix_lens; tp.n_seg = n_groups;
    tp.status = status;
    // upper bound of the groups' row tiles (each group rounds up once)
    const int64_t tiles = ((int64_t)n_req * G +
                           (int64_t)(TILE_ROWS - 1) * (n_groups < n_req ? n_groups : n_req)) /
                          TILE_ROWS;
    tp.part_rows = (int64_t)n_req * n_kv * G;
    // (one part more for the requests' own keys)
    const int64_t part_floats = tp.part_rows * (PR_HD + 2);
    tp.parts = parts_for(tiles * n_kv, bt_width, part_floats, scratch_floats - part_floats);
    tp.parts_out = scratch;
    tp.parts_ml = scratch + (tp.parts + 1) * tp.part_rows * PR_HD;
    p.max_rows = FEW_ROWS;
    p.beside = 1;
    p.part = tp.parts; p.part_rows = tp.part_rows;
    p.parts_o = tp.parts_out; p.parts_ml = tp.parts_ml;
    int rc2 = launch_tile_attn(who, tp, (int)tiles, (int)tiles, n_req, s);
    if (rc2 == LOCKS_OK) rc2 = launch_row_attn(who, p, n_req, G, 1, s);
    if (rc2 == LOCKS_OK) rc2 = launch_join_parts(who, tp, tp.parts + 1, n_req, s);
    return rc2;
}
