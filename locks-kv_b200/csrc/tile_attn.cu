// Paged attention of many query rows at a time on the 5th-generation tensor cores:
// the prompt (and long-chunk) half of the windowed attention, and the shared part of
// the shared-prefix decode.
//
// A "segment" is a run of query tokens that read one table row: a request's new
// tokens, or the single tokens of the requests that share a prefix.  Its rows
// (token, query head of the KV head) are packed, row = token * G + head, and cut
// into tiles of up to 256.  A work item is a tile of one KV head (and one part of its
// keys); it walks the pages the tile can see -- first pages and recent ones as one
// list -- eight pages = 128 keys at a time:
//
//   S [128 rows x 128 keys] = Q K^T       tcgen05.mma, Q and K in shared memory
//   P = exp2(scale (S - m)), l += sum P   a thread per row: its row of S comes from
//                                         tensor memory, P goes back there in bf16
//   O [128 rows x 128] += P V             tcgen05.mma, A = P from tensor memory
//
// Two such streams run against each other, so that one's softmax hides behind the
// other's products.  With more than 128 rows each stream has 128 of them and both
// walk every key tile; with fewer, both have the same rows and take the key tiles in
// turn (joined at the end: both O are in the same tensor-memory lanes): a decode batch
// is then not half idle.
//
// One CTA per SM works through its share of the items; every stage runs ahead of the
// next one across item borders, so that an item's start (finding it, Q, the first
// pages: about 8 us when nothing overlaps it) and its end hide behind its neighbours.
// Warps 0-3 and 4-7: softmax of stream 0 and 1 (thread = row = tensor-memory lane).
// Warp 8: one thread issues all products.  Warp 9: fetches pages through the table by
// tiled tensor-map copies into a ring of four 32 KiB tiles that K and V share.
// Warp 10: finds the items.  Warp 11: Q.
// Tensor memory: S / P of the streams in columns 0 and 128, O in 256 and 384.
//
// The running maximum is only raised when it grows by more than 2^8 (O and l then get
// rescaled): P stays below 2^8 and no row of O is touched in most steps.  P is rounded to
// bf16 because V is (both operands of the product have one type), half a step each; m, l,
// S and O are fp32.  (A second product with what the rounding left would take half again
// as much of the tensor pipe, 63 % busy in a prompt, and twice the stores of P.)
//
// Every wait is bounded (status word; later waits then return at once, work and copies
// in flight are waited for and tensor memory is freed).  No multicast.
#include "common.cuh"
#include "paged_rows.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace locks {
namespace {

constexpr int TA_THREADS = 384;
constexpr int TA_RING = 4;
constexpr int TA_TILE = 128;                       // keys of a tile, rows of a stream
constexpr int TA_PAGES = TA_TILE / PR_PAGE;
constexpr int TA_HALF = TA_TILE * 128;             // bytes: 128 rows x 64 channels
constexpr int TA_BYTES = 2 * TA_HALF;
constexpr int TA_BOX = PR_PAGE * 256;              // bytes of a page of one plane and head
constexpr int TM_S = 0, TM_O = 256, TM_COLS = 512;
constexpr float TA_RAISE = 8.f;
// one pair of exponentials in TA_POLY leaves the special-function unit alone
constexpr int TA_POLY = 4;
// P is handed over in two steps, so that the product of the first is under way while
// the exponentials of the second are taken
constexpr int TA_EARLY = 4;                        // pages (k-steps) of the first step

struct Item {
    int valid, kh, part, t0, row0, n_rows, j0, n_tiles, key_end, written, base_pos;
    int table_row;
    PageList list;
};

struct __align__(1024) TileSmem {
    uint8_t q[2][TA_BYTES];
    uint8_t ring[TA_RING][TA_BYTES];
    uint8_t stage[8][4096];                        // a softmax warp's way out: 32 rows x 128 B
    uint64_t full[TA_RING], empty[TA_RING], tail, drain;
    uint64_t item_full[2], item_empty[2], q_full[2], q_empty;
    uint64_t s_full[2], p_early[2], p_ready[2], o_full[2], meet;
    Item item[2];
    uint32_t tmem_base;
    int dead;
};
static_assert(sizeof(TileSmem) + 1024 <= 232448, "one CTA's shared memory");
constexpr int TA_READERS = 11;                     // warps that read an item: all but its finder

// maxima that a NaN goes through
__device__ __forceinline__ float max2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
          "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}

// 2^x of a pair on the multiply-add pipe, x <= 127: 2^n 2^f with n the nearest whole
// number (read off the low bits of x + 1.5 2^23) and 1 + f q(f), |f| <= 1/2, q of degree
// 3 (own minimax fit, relative error 2.8e-6: P is rounded to 8 bits anyway, and the
// sum's error stays below that).  Below -127, where a hidden key's -inf lands, it is
// exactly 0, because the polynomial is exactly 1 at f = 0.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 t = add2(x, make_float2(12582912.f, 12582912.f));
    const float2 n = add2(t, make_float2(-12582912.f, -12582912.f));
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 r = make_float2(0x1.3a02ccp-7f, 0x1.3a02ccp-7f);
    r = fma2(r, f, make_float2(0x1.c9fc46p-5f, 0x1.c9fc46p-5f));
    r = fma2(r, f, make_float2(0x1.ec0378p-3f, 0x1.ec0378p-3f));
    r = fma2(r, f, make_float2(0x1.62e12cp-1f, 0x1.62e12cp-1f));
    r = fma2(r, f, make_float2(1.f, 1.f));
    r.x = __int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23));
    r.y = __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23));
    return r;
}

// a wait that gives up once any wait of the CTA has
__device__ __forceinline__ bool is_dead(TileSmem& sm) {
    return *reinterpret_cast<volatile int*>(&sm.dead) != 0;
}
__device__ __forceinline__ void ta_wait(TileSmem& sm, uint64_t* bar, uint32_t parity,
                                        int* status) {
    if (!mbar_try_wait(bar, parity)) {
        bool ok = false;
        for (int it = 0; it < (1 << 22) && !ok; ++it) {
            ok = mbar_try_wait(bar, parity);
            if (!ok && it > 64) {
                __nanosleep(32);
                if (is_dead(sm)) break;
            }
        }
        if (!ok && !is_dead(sm)) {
            *reinterpret_cast<volatile int*>(&sm.dead) = 1;
            if (status) atomicExch(status, LOCKS_ST_WAIT_TIMEOUT);
        }
    }
    __syncwarp();
}

// 16 bytes global -> shared; src_bytes 0: zeros, nothing is read
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// One box = one page of a head: [token / 8][channel / 64][token % 8][64 channels], so
// that a tile of pages has its groups of 8 keys 2 KiB apart throughout (one box per page
// instead of one per 64 channels: the copy engine takes about 35 ns for a box of either
// size, and the tile loop would wait for it).
__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int chunk,
                                              int block, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %2, %3, %2, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(0), "r"(chunk), "r"(block), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* map, int channel,
                                              int head, int token, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(channel), "r"(head), "r"(token), "r"(smem_u32(bar))
        : "memory");
}

// segment s: first token and token count (0 where the few-row kernel serves it)
__device__ __forceinline__ void segment(const TileAttnParams& p, int s, int& t0, int& n) {
    t0 = p.bounds[s];
    n = min(p.bounds[s + 1], p.r.n_tok) - t0;
    if (t0 < 0 || (!p.prefix_lens && n * p.r.G <= p.min_rows)) n = 0;
    n = max(n, 0);
}
__device__ __forceinline__ int tiles_of(const TileAttnParams& p, int n) {
    return (n * p.r.G + 2 * TA_TILE - 1) / (2 * TA_TILE);
}

// tiles of all segments, by one warp
__device__ __forceinline__ int count_tiles(const TileAttnParams& p, int lane) {
    int sum = 0;
#pragma unroll 4
    for (int s = lane; s < p.n_seg; s += 32) {
        int t0, n;
        segment(p, s, t0, n);
        sum += tiles_of(p, n);
    }
    return __reduce_add_sync(0xffffffffu, sum);
}

// Where a search for tiles stands: segments from s0 on begin with tile number `before`.
struct FindState {
    int s0, before;
};

// Row tile `target` with KV head and part `rest`, by one warp; false: there is no such
// tile (the tiles were not counted).
__device__ __forceinline__ bool find_item(const TileAttnParams& p, int target, int rest,
                                          int lane, FindState& at, Item& it) {
    if (target < at.before) at = {0, 0};
    for (; at.s0 < p.n_seg; at.s0 += 32) {
        const int s0 = at.s0, before = at.before;
        int t0 = 0, n = 0, extent = 0, end = 0;
        if (s0 + lane < p.n_seg) {
            extent = p.prefix_lens ? p.prefix_lens[s0 + lane] : p.r.seq_lens[s0 + lane];
            segment(p, s0 + lane, t0, n);
            end = p.bounds[s0 + lane + 1];
        }
        const int mine = tiles_of(p, n);
        int x = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        const int from = before + x - mine;
        const uint32_t hit = __ballot_sync(0xffffffffu, target >= from && target < from + mine);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.t0 = __shfl_sync(0xffffffffu, t0, src);
            n = __shfl_sync(0xffffffffu, n, src);
            extent = __shfl_sync(0xffffffffu, extent, src);
            // longest rows first
            const int tile = __shfl_sync(0xffffffffu, mine - 1 - (target - from), src);
            const int G = p.r.G;
            it.kh = rest % p.r.n_kv;
            it.part = rest / p.r.n_kv;
            it.row0 = tile * 2 * TA_TILE;
            it.n_rows = min(n * G - it.row0, 2 * TA_TILE);
            it.base_pos = 0;
            if (p.prefix_lens) {
                const int whole = min(max(extent, 0) / PR_PAGE, p.r.bt_width);
                it.written = it.key_end = whole * PR_PAGE;
                it.table_row = it.t0;
                it.list = page_list(0, it.key_end - 1, INT32_MAX, 0, p.r.bt_width);
            } else {
                it.written = extent;
                // (where the queries sit goes by the bounds, cut off or not)
                it.base_pos = it.written - (__shfl_sync(0xffffffffu, end, src) - it.t0);
                it.table_row = s0 + src;
                it.list = page_list(it.base_pos + it.row0 / G,
                                    it.base_pos + (it.row0 + it.n_rows - 1) / G, p.r.window,
                                    p.r.sinks, p.r.bt_width);
                it.key_end = it.list.key_end;
            }
            const int all = (it.list.n + TA_PAGES - 1) / TA_PAGES;
            const int per = (all + p.parts - 1) / p.parts;
            it.j0 = min(it.part * per, all);
            it.n_tiles = min(it.j0 + per, all) - it.j0;
            it.valid = 1;
            return true;
        }
        at.before += __shfl_sync(0xffffffffu, x, 31);
    }
    return false;
}

__global__ void __launch_bounds__(TA_THREADS, 1)
tile_attn_kernel(const __grid_constant__ CUtensorMap map_q,
                 const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const TileAttnParams p) {
    extern __shared__ uint8_t ta_raw[];
    TileSmem& sm = *reinterpret_cast<TileSmem*>(
        ta_raw + ((1024u - (smem_u32(ta_raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x, lane = tid & 31, G = p.r.G;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // uniform, and known to be

    // ---- setup -------------------------------------------------------------------
    if (tid == 0) {
        sm.dead = 0;
        for (int i = 0; i < TA_RING; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
        mbar_init(&sm.tail, 1);
        mbar_init(&sm.drain, 1);
        mbar_init(&sm.meet, 8);
        mbar_init(&sm.q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], TA_READERS);
            mbar_init(&sm.q_full[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_early[i], 4);
            mbar_init(&sm.p_ready[i], 4);
            mbar_init(&sm.o_full[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sm.tmem_base)), "r"(TM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before_sync();
    }
    // everything before this launch is done; the call's next launch may take SMs as they
    // free up
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = sm.tmem_base;

    // the n-th item of this CTA: null when there is none (or a wait ran out)
    auto next_item = [&](int n) -> const Item* {
        ta_wait(sm, &sm.item_full[n & 1], (uint32_t)(n >> 1) & 1u, p.status);
        if (__any_sync(0xffffffffu, is_dead(sm))) return nullptr;
        return sm.item[n & 1].valid ? &sm.item[n & 1] : nullptr;
    };
    auto done_with = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[n & 1]);
    };

    // registers: 12 warps start with 168 each; the softmax threads hold a row of S
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 10) {
            // ---- items ----------------------------------------------------------------
            // (tiles fastest; those nobody expects come behind all the others)
            const int tiles = p.tile_bound ? p.tile_bound : count_tiles(p, lane);
            const int expected = tiles * p.r.n_kv * p.parts;
            const int total = expected + p.tile_more * p.r.n_kv * p.parts;
            FindState at = {0, 0};
            int n = 0;
            for (int w = blockIdx.x; !__any_sync(0xffffffffu, is_dead(sm)); w += gridDim.x) {
                Item it;
                it.valid = 0;
                if (w < total) {
                    const int n_tiles = w < expected ? tiles : p.tile_more;
                    const int x = w < expected ? w : w - expected, rest = x / n_tiles;
                    const int target = x - rest * n_tiles + (w < expected ? 0 : tiles);
                    if (!find_item(p, target, rest, lane, at, it)) continue;
                }
                if (n >= 2)
                    ta_wait(sm, &sm.item_empty[n & 1], (uint32_t)((n >> 1) - 1) & 1u, p.status);
                if (lane == 0) {
                    sm.item[n & 1] = it;
                    mbar_arrive(&sm.item_full[n & 1]);
                }
                __syncwarp();
                ++n;
                if (!it.valid) break;
            }
        } else if (warp == 11) {
            // ---- Q into the swizzled K-major layout, 16 lanes to a row -------------------
            int loads = 0, both = 0;
            for (int n = 0;; ++n) {
                const Item* item = next_item(n);
                if (!item) break;
                const int row0 = item->row0, n_rows = item->n_rows, t0 = item->t0,
                          kh = item->kh, n_tiles = item->n_tiles;
                done_with(n);
                if (n_tiles == 0) continue;
                if (loads > 0) {
                    ta_wait(sm, &sm.q_empty, (uint32_t)(loads - 1) & 1u, p.status);
                    if (__any_sync(0xffffffffu, is_dead(sm))) break;    // Q is in use still
                }
                ++loads;
                const int subs = n_rows > TA_TILE ? 2 : 1;
                both += subs - 1;
                if (TA_TILE % G == 0) {
                    // a stream's rows are whole tokens: one box for each half of the
                    // channels (rows behind the last one are somebody else's or zeros:
                    // a row only reaches its own output, which is not stored)
                    if (lane == 0)
                        for (int sub = 0; sub < subs; ++sub) {
                            mbar_expect_tx(&sm.q_full[sub], TA_BYTES);
                            for (int half = 0; half < 2; ++half)
                                tma_load_rows(&sm.q[sub][half * TA_HALF], &map_q, 64 * half, kh * G,
                                              t0 + (row0 + sub * TA_TILE) / G, &sm.q_full[sub]);
                        }
                    __syncwarp();
                    continue;
                }
                // (rows behind the last one are zeros; every copy is on its way before
                // the first is waited for)
                const int piece = lane & 15;
                int row = lane >> 4, tok = (row0 + row) / G, g = row0 + row - tok * G;
                const __nv_bfloat16* src = p.r.q + (int64_t)(t0 + tok) * p.r.q_tok +
                                           (int64_t)(kh * G + g) * p.r.q_head + 8 * piece;
                // two rows on: in the same token, or in the next one
                const int64_t stay = 2 * p.r.q_head, wrap = p.r.q_tok + (2 - G) * p.r.q_head;
                const uint32_t d0 = smem_u32(sm.q) + (piece >> 3) * TA_HALF;
                for (int sub = 0; sub < subs; ++sub) {
#pragma unroll 8
                    for (int k = 0; k < TA_TILE / 2; ++k) {
                        const bool live = row < n_rows;
                        const int r = row & (TA_TILE - 1);
                        cp_async16(d0 + sub * TA_BYTES + r * 128 + ((piece ^ r) & 7) * 16,
                                   live ? src : p.r.q, live ? 16 : 0);
                        const bool over = g + 2 >= G;
                        src += over ? wrap : stay;
                        g += 2 - (over ? G : 0);
                        row += 2;
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.q_full[sub]);
                }
            }
            if (__any_sync(0xffffffffu, is_dead(sm))) {     // copies in flight land first
                if (loads > 0) mbar_wait(&sm.q_full[0], (uint32_t)(loads - 1) & 1u, p.status);
                if (both > 0) mbar_wait(&sm.q_full[1], (uint32_t)(both - 1) & 1u, p.status);
            }
        } else if (warp == 9) {
            // ---- pages: K and V tiles in the order the products take them ---------------
            int slot = 0, issued = 0, cuts = 0;
            for (int n = 0;; ++n) {
                const Item* item = next_item(n);
                if (!item) break;
                const PageList list = item->list;
                const int j0 = item->j0, n_tiles = item->n_tiles, written = item->written;
                const int chunk = item->kh * p.head_chunks;
                const bool by_rows = item->n_rows > TA_TILE;
                const int32_t* table = p.r.table + (int64_t)item->table_row * p.r.bt_stride;
                done_with(n);
                auto fetch = [&](int j, bool is_v) {
                    const int v = (j0 + j) * TA_PAGES + (lane & 7);
                    int blk = p.r.num_blocks;           // outside the map: zeros
                    bool partial = false;
                    int page = 0;
                    if (v < list.n) {
                        page = list.page(v);
                        blk = min(max(table[page], 0), p.r.num_blocks - 1);
                        partial = is_v && (page + 1) * PR_PAGE > written;
                    }
                    if (issued >= TA_RING)
                        ta_wait(sm, &sm.empty[slot], (uint32_t)((issued / TA_RING) - 1) & 1u,
                                p.status);
                    if (__any_sync(0xffffffffu, is_dead(sm))) return;
                    const uint32_t cut = __ballot_sync(0xffffffffu, lane < 8 && partial);
                    uint64_t* bar = cut ? &sm.tail : &sm.full[slot];
                    if (lane == 0) mbar_expect_tx(bar, TA_BYTES);
                    __syncwarp();
                    if (lane < TA_PAGES)
                        tma_load_page(&sm.ring[slot][lane * TA_BOX], is_v ? &map_v : &map_k,
                                      chunk, blk, bar);
                    if (cut) {
                        // the sequence ends inside a page: what the cache holds behind it
                        // may be anything, and 0 x NaN is not 0
                        ta_wait(sm, &sm.tail, (uint32_t)cuts & 1u, p.status);
                        ++cuts;
                        const int s = __ffs(cut) - 1;
                        const int from =
                            max(written - __shfl_sync(0xffffffffu, page, s) * PR_PAGE, 0);
                        for (int e = lane; e < (PR_PAGE - from) * 16; e += 32)
                            *reinterpret_cast<uint4*>(
                                &sm.ring[slot][s * TA_BOX + ((from + (e >> 4)) >> 3) * 2048 +
                                               ((e >> 3) & 1) * 1024 +
                                               ((from + (e >> 4)) & 7) * 128 + (e & 7) * 16]) =
                                make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.full[slot]);
                    }
                    slot = slot + 1 == TA_RING ? 0 : slot + 1;
                    ++issued;
                };
                if (n_tiles > 0) fetch(0, false);
                if (!by_rows && n_tiles > 1) fetch(1, false);
                for (int j = 0; j < n_tiles; ++j) {
                    fetch(j, true);
                    const int next = by_rows ? j + 1 : j + 2;
                    if (next < n_tiles) fetch(next, false);
                }
            }
            // a wait ran out: nobody consumed the last copies; they must land all the same
            // (those of a tile with a cut page complete on `tail`, and only the last such
            // tile's can be under way)
            if (__any_sync(0xffffffffu, is_dead(sm)))
                for (int i = max(issued - TA_RING, 0); i < issued + min(cuts, 1); ++i)
                    mbar_wait(i < issued ? &sm.full[i % TA_RING] : &sm.tail,
                              (uint32_t)(i < issued ? i / TA_RING : cuts - 1) & 1u, p.status);
        } else if (warp == 8) {
            // ---- products -------------------------------------------------------------
            constexpr uint32_t ID_S = tc_idesc(TA_TILE, false), ID_O = tc_idesc(PR_HD, true);
            const uint64_t desc_q = tc_desc(smem_u32(sm.q), 16, 1024),
                           desc_k = tc_desc(smem_u32(sm.ring), 16, 2048),
                           desc_v = tc_desc(smem_u32(sm.ring), 1024, 2048);
            int slot = 0, taken = 0, loads = 0, both = 0;
            uint32_t phase[2] = {0, 0};             // tiles of each stream, over all items
            auto take = [&]() {                     // the next tile of the ring
                const int s = slot;
                ta_wait(sm, &sm.full[s], (uint32_t)(taken / TA_RING) & 1u, p.status);
                slot = slot + 1 == TA_RING ? 0 : slot + 1;
                ++taken;
                return s;
            };
            auto commit = [&](uint64_t* bar) {
                if (tc_elect()) tc_commit(bar);
                __syncwarp();
            };
            for (int n = 0;; ++n) {
                const Item* item = next_item(n);
                if (!item) break;
                const int n_tiles = item->n_tiles;
                const bool by_rows = item->n_rows > TA_TILE;
                done_with(n);
                if (n_tiles == 0) continue;
                auto scores = [&](int i, int s) {
                    tc_after_sync();
                    const uint64_t a = desc_q + (uint64_t)((by_rows ? i : 0) * (TA_BYTES >> 4));
                    const uint64_t b = desc_k + (uint64_t)(s * (TA_BYTES >> 4));
                    if (tc_elect()) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint64_t in_row = (ks & 3) * 32 >> 4, half = ks >> 2;
                            tc_mma_ss(tmem + TM_S + i * TA_TILE,
                                      a + in_row + half * (TA_HALF >> 4),
                                      b + in_row + half * (1024 >> 4), ID_S, ks ? 1u : 0u);
                        }
                        tc_commit(&sm.s_full[i]);
                    }
                    __syncwarp();
                };
                auto values = [&](int i, int s, int t) {    // the item's tile t of stream i
                    const uint64_t b = desc_v + (uint64_t)(s * (TA_BYTES >> 4));
                    const uint32_t par = phase[i]++ & 1u;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        ta_wait(sm, half ? &sm.p_ready[i] : &sm.p_early[i], par, p.status);
                        tc_after_sync();
                        if (tc_elect()) {
#pragma unroll
                            for (int ks = half ? TA_EARLY : 0; ks < (half ? TA_PAGES : TA_EARLY);
                                 ++ks)
                                tc_mma_ts(tmem + TM_O + i * PR_HD, tmem + TM_S + i * TA_TILE + ks * 8,
                                          b + (uint64_t)((ks * TA_BOX) >> 4), ID_O,
                                          (t | ks) ? 1u : 0u);
                            if (half) tc_commit(&sm.o_full[i]);
                        }
                        __syncwarp();
                    }
                };
                int k_slot = take();
                ta_wait(sm, &sm.q_full[0], (uint32_t)loads & 1u, p.status);
                ++loads;
                scores(0, k_slot);
                if (by_rows) {
                    ta_wait(sm, &sm.q_full[1], (uint32_t)both & 1u, p.status);
                    ++both;
                    scores(1, k_slot);
                    commit(&sm.empty[k_slot]);
                    if (n_tiles == 1) commit(&sm.q_empty);
                    // (the ring's next tiles are waited for while products run)
                    int v_slot = take();
                    for (int j = 0; j < n_tiles; ++j) {
                        const bool more = j + 1 < n_tiles;
                        if (more) k_slot = take();
                        values(0, v_slot, j);
                        if (more) scores(0, k_slot);
                        values(1, v_slot, j);
                        commit(&sm.empty[v_slot]);
                        if (more) {
                            scores(1, k_slot);
                            commit(&sm.empty[k_slot]);
                            if (j + 2 == n_tiles) commit(&sm.q_empty);
                            v_slot = take();
                        }
                    }
                } else {
                    commit(&sm.empty[k_slot]);
                    if (n_tiles > 1) {
                        k_slot = take();
                        scores(1, k_slot);
                        commit(&sm.empty[k_slot]);
                    }
                    if (n_tiles <= 2) commit(&sm.q_empty);
                    for (int j = 0; j < n_tiles; ++j) {
                        const int v_slot = take();
                        values(j & 1, v_slot, j >> 1);
                        commit(&sm.empty[v_slot]);
                        if (j + 2 < n_tiles) {
                            k_slot = take();
                            scores(j & 1, k_slot);
                            commit(&sm.empty[k_slot]);
                            if (j + 3 == n_tiles) commit(&sm.q_empty);
                        }
                    }
                }
            }
            if (__any_sync(0xffffffffu, is_dead(sm))) {     // products in flight end first
                commit(&sm.drain);
                mbar_wait(&sm.drain, 0, p.status);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: stream i, thread = row ---------------------------------------
        const int i = warp >> 2, q4 = warp & 3;
        const uint32_t lane_base = tmem + ((uint32_t)(q4 * 32) << 16);
        const uint32_t ts = lane_base + TM_S + i * TA_TILE;
        const float sl2 = p.r.scale_log2;
        uint32_t phase = 0;                         // tiles of this stream, over all items
        uint32_t meetings = 0;
        auto meet = [&]() {                         // all eight softmax warps (bounded too)
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.meet);
            ta_wait(sm, &sm.meet, meetings++ & 1u, p.status);
        };
        for (int n = 0;; ++n) {
            const Item* item = next_item(n);
            if (!item) break;
            const PageList list = item->list;
            const int j0 = item->j0, n_tiles = item->n_tiles, n_rows = item->n_rows;
            const bool by_rows = n_rows > TA_TILE;
            const int local = (by_rows ? i * TA_TILE : 0) + q4 * 32 + lane;
            const int row = item->row0 + min(local, n_rows - 1);
            const int t0 = item->t0, tok = row / G, head = item->kh * G + row - tok * G;
            const int pos = p.prefix_lens ? p.r.seq_lens[t0 + tok] - 1 : item->base_pos + tok;
            const int last_key = min(pos, item->key_end - 1), part = item->part;
            done_with(n);
            const int first_key = pos >= p.r.window ? pos - p.r.window + 1 : 0;
            const int sinks = p.r.sinks;
            // (row order is position order only for a request's own tokens)
            const int w_last = __reduce_min_sync(0xffffffffu, last_key);
            const int w_first = __reduce_max_sync(0xffffffffu, first_key);
            // tiles [clear_lo, clear_hi) hide no key from any row of the warp: keys up to
            // the oldest row's, and either all first keys or all in the newest's window
            int clear_lo, clear_hi;
            {
                const int n_win = max(w_last + 1, 0) / PR_PAGE - list.shift;    // entries before it
                clear_hi = min(list.n, n_win) / TA_PAGES;
                const int sink_hi = min(min(list.n_first, sinks / PR_PAGE),
                                        max(w_last + 1, 0) / PR_PAGE) / TA_PAGES;
                const int from = max((w_first + PR_PAGE - 1) / PR_PAGE - list.shift,
                                     list.shift > 0 && w_first > 0 ? list.n_first : 0);
                clear_lo = (from + TA_PAGES - 1) / TA_PAGES;
                if (clear_hi <= clear_lo) { clear_lo = 0; clear_hi = sink_hi; }
            }
            float m = -INFINITY, l = 0.f;
            int t = 0;                              // this item's tiles of this stream so far
            for (int j = by_rows ? 0 : i; j < n_tiles; j += by_rows ? 1 : 2, ++t, ++phase) {
                ta_wait(sm, &sm.s_full[i], phase & 1u, p.status);
                tc_after_sync();
                uint32_t sr[TA_TILE];
                float* s = reinterpret_cast<float*>(sr);
                float mx[8];
                auto peaks = [&](int c0) {          // maxima of columns c0 .. c0 + 63
#pragma unroll
                    for (int c = c0; c < c0 + 64; c += 16)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            mx[e] = c == 0 ? max2(s[e], s[8 + e]) : max3(mx[e], s[c + e], s[c + 8 + e]);
                };
                tc_ld32(ts, sr);
                tc_ld32(ts + 32, sr + 32);
                tc_wait_ld();
                tc_tie32(sr);
                tc_tie32(sr + 32);
                tc_ld32(ts + 64, sr + 64);
                tc_ld32(ts + 96, sr + 96);
                const int jt = j0 + j;
                if (jt >= clear_lo && jt < clear_hi) {
                    peaks(0);
                    tc_wait_ld();
                    tc_tie32(sr + 64);
                    tc_tie32(sr + 96);
                    peaks(64);
                } else {
                    tc_wait_ld();
                    tc_tie32(sr + 64);
                    tc_tie32(sr + 96);
                    const int v0 = jt * TA_PAGES;
#pragma unroll
                    for (int pg = 0; pg < TA_PAGES; ++pg) {
                        uint32_t keep = 0;
                        if (v0 + pg < list.n) {
                            const int base = list.page(v0 + pg) * PR_PAGE;
                            const int hi = last_key - base, lo = first_key - base,
                                      sk = sinks - base;
                            const uint32_t m_hi = hi < 0 ? 0u : hi > 15 ? 0xFFFFu : (2u << hi) - 1u;
                            const uint32_t m_lo = lo <= 0 ? 0xFFFFu : lo > 15 ? 0u : 0xFFFFu << lo;
                            const uint32_t m_sk = sk <= 0 ? 0u : sk > 15 ? 0xFFFFu : (1u << sk) - 1u;
                            keep = m_hi & (m_lo | m_sk);
                        }
#pragma unroll
                        for (int c = 0; c < PR_PAGE; ++c)
                            if (!(keep >> c & 1u)) s[pg * PR_PAGE + c] = -INFINITY;
                    }
                    peaks(0);
                    peaks(64);
                }
                const float tile_max = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]),
                                            max2(mx[6], mx[7]));
                if (t == 0) {
                    m = tile_max;
                } else if (__any_sync(0xffffffffu, (tile_max - m) * sl2 > TA_RAISE)) {
                    // (m -inf: nothing seen so far, O and l are 0 and stay it)
                    const float up = fmaxf(m, tile_max);
                    const float f = m == -INFINITY ? 0.f : pr_exp2((m - up) * sl2);
                    m = up;
                    l *= f;
                    ta_wait(sm, &sm.o_full[i], (phase - 1) & 1u, p.status);
                    tc_after_sync();
                    const uint32_t to = lane_base + TM_O + i * PR_HD;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[16];
                        tc_ld16(to + 16 * c, o);
                        tc_wait_ld();
                        tc_tie16(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tc_st16(to + 16 * c, o);
                    }
                }
                // A score of NaN or +inf makes the row NaN: its maximum becomes NaN, with
                // it every exponent, and so l and O (three of four exponentials are the
                // special-function unit's; the polynomial turns NaN into 0)
                if (tile_max != tile_max) m = tile_max;
                const float ml2 = m * sl2;
                const float base = m == -INFINITY ? 0.f : fmaf(ml2, 0.f, ml2);
                const float2 k2 = make_float2(sl2, sl2), b2 = make_float2(-base, -base);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 x = fma2(make_float2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), k2, b2);
                        if (e % TA_POLY == TA_POLY - 1) {
                            x = exp2_poly(x);
                        } else {
                            x.x = pr_exp2(x.x);
                            x.y = pr_exp2(x.y);
                        }
                        sum[e & 1] = add2(sum[e & 1], x);
                        pk[e] = pack_bf16x2(x.x, x.y);
                    }
                    tc_st16(ts + 16 * c, pk);
                    if (2 * (c + 1) == TA_EARLY || c == 3) {
                        tc_wait_st();
                        tc_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(c == 3 ? &sm.p_ready[i] : &sm.p_early[i]);
                    }
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            // ---- results: columns [from, from + 32 chunks) of O ---------------------------
            if (t > 0) {
                ta_wait(sm, &sm.o_full[i], (phase - 1) & 1u, p.status);
                tc_after_sync();
            }
            // streams that share the rows: each finishes half of the channels
            const int chunk0 = by_rows ? 0 : 2 * i, chunks = by_rows ? 4 : 2;
            // (a sum that is NaN is not zero: the row is NaN, not one that saw nothing)
            float w_mine = l != 0.f ? 1.f : 0.f, w_other = 0.f;
            if (!by_rows) {
                float2* mine = reinterpret_cast<float2*>(sm.stage[warp]) + lane;
                *mine = make_float2(m, l);
                tc_before_sync();
                meet();
                tc_after_sync();
                const float2 other = reinterpret_cast<float2*>(sm.stage[warp ^ 4])[lane];
                meet();
                const float m1 = other.x, l1 = other.y;
                const float up = fmaxf(m, m1);
                w_mine = l != 0.f ? pr_exp2((m - up) * sl2) : 0.f;
                w_other = l1 != 0.f ? pr_exp2((m1 - up) * sl2) : 0.f;
                l = w_mine * l + w_other * l1;
                m = up;
            }
            const bool final = p.parts_out == nullptr;
            const float inv = !final ? 1.f : l != 0.f ? 1.f / l : 0.f;
            w_mine *= inv;
            w_other *= inv;
            const int64_t part_at = (int64_t)part * p.part_rows +
                                    (int64_t)(t0 + tok) * p.r.n_kv * G + head;
            // a row's way out: through the warp's stage, 128 B of every row at a time, so
            // that the stores are whole lines
            const int64_t my_off = final ? ((int64_t)(t0 + tok) * p.r.o_tok +
                                            (int64_t)head * p.r.o_head) * 2
                                         : part_at * (PR_HD * 4);
            uint8_t* dst = final ? reinterpret_cast<uint8_t*>(p.r.out)
                                 : reinterpret_cast<uint8_t*>(p.parts_out);
            const bool any = __any_sync(0xffffffffu, l != 0.f);
            uint8_t* stage = sm.stage[warp];
            const int live = min(n_rows - (by_rows ? i * TA_TILE : 0) - q4 * 32, 32);
            int64_t off[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                off[k] = __shfl_sync(0xffffffffu, my_off, 4 * k + (lane >> 3)) + 16 * (lane & 7);
            auto send = [&](int byte) {             // bytes [byte, byte + 128) of the rows
                __syncwarp();
                uint4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    x[k] = *reinterpret_cast<const uint4*>(
                        stage + tc_swz(4 * k + (lane >> 3), 16 * (lane & 7)));
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (4 * k + (lane >> 3) < live)
                        *reinterpret_cast<uint4*>(dst + off[k] + byte) = x[k];
                __syncwarp();
            };
            // 128 columns of tensor memory: all of this stream's O, or the same 64 of both
            uint32_t o[TA_TILE];
            float* f = reinterpret_cast<float*>(o);
            if (final || any) {
                const uint32_t here = lane_base + TM_O + i * PR_HD + 32 * chunk0;
                const uint32_t there =
                    by_rows ? here + 64 : lane_base + TM_O + (1 - i) * PR_HD + 32 * chunk0;
                tc_ld32(here, o);
                tc_ld32(here + 32, o + 32);
                tc_ld32(there, o + 64);
                tc_ld32(there + 32, o + 96);
                tc_wait_ld();
                tc_tie32(o);
                tc_tie32(o + 32);
                tc_tie32(o + 64);
                tc_tie32(o + 96);
                // (without a product there is no O)
                const float w2 = by_rows ? w_mine : w_other;
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    f[e] = w_mine != 0.f ? w_mine * f[e] : 0.f;
                    f[64 + e] = w2 != 0.f ? w2 * f[64 + e] : 0.f;
                }
                if (!by_rows)
#pragma unroll
                    for (int e = 0; e < 64; ++e) f[e] += f[64 + e];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c >= chunks) break;
                    if (final) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            *reinterpret_cast<uint4*>(stage + tc_swz(lane, (c & 1) * 64 + 2 * e)) =
                                make_uint4(pack_bf16x2(f[32 * c + e], f[32 * c + e + 1]),
                                           pack_bf16x2(f[32 * c + e + 2], f[32 * c + e + 3]),
                                           pack_bf16x2(f[32 * c + e + 4], f[32 * c + e + 5]),
                                           pack_bf16x2(f[32 * c + e + 6], f[32 * c + e + 7]));
                        if (c & 1) send(((chunk0 + c) >> 1) * 128);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(stage + tc_swz(lane, 4 * e)) =
                                make_float4(f[32 * c + e], f[32 * c + e + 1], f[32 * c + e + 2],
                                            f[32 * c + e + 3]);
                        send((chunk0 + c) * 128);
                    }
                }
            }
            if (local < n_rows && (by_rows || i == 0)) {
                if (!final)         // O is relative to m; (m in log2 units, l)
                    *reinterpret_cast<float2*>(p.parts_ml + 2 * part_at) =
                        make_float2(l != 0.f ? m * sl2 : -INFINITY, l);
                else if (p.r.lse)
                    p.r.lse[(int64_t)(t0 + tok) * p.r.lse_tok + head] =
                        l != 0.f ? (m * sl2 + log2f(l)) * PR_LN2 : -INFINITY;
            }
            tc_before_sync();
            // (the other stream has read this one's O and sums before they change)
            if (!by_rows) meet();
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 8) {
        tc_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     ::"r"(tmem), "r"(TM_COLS) : "memory");
    }
}

// A cache plane as (64 channels, 8 tokens, chunks of 64 channels, token groups of a
// page, blocks): a head is two chunks, `sh / 64` chunks from the next head
CUresult encode_plane(CUtensorMap* map, const void* base, int n_kv, int num_blocks,
                      int64_t sh, int64_t st, int64_t sb) {
    EncodeTiledFn enc = encode_tiled();
    if (enc == nullptr) return CUDA_ERROR_NOT_SUPPORTED;
    const int64_t chunks = (n_kv - 1) * (sh / 64) + 2;
    const cuuint64_t dim[5] = {64, 8, (cuuint64_t)chunks, 2, (cuuint64_t)num_blocks};
    // (a dimension of one may come with any stride)
    const cuuint64_t stride[4] = {(cuuint64_t)st * 2, 128, (cuuint64_t)st * 16,
                                  (cuuint64_t)(num_blocks > 1 ? sb : PR_PAGE * st) * 2};
    const cuuint32_t box[5] = {64, 8, 2, 2, 1}, one[5] = {1, 1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dim, stride,
               box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Q as (128 channels, heads, tokens), boxes of 64 channels x the G heads of a KV head x
// the tokens of 128 rows
CUresult encode_q(CUtensorMap* map, const RowAttnParams& r, int n_tok) {
    EncodeTiledFn enc = encode_tiled();
    if (enc == nullptr) return CUDA_ERROR_NOT_SUPPORTED;
    const cuuint64_t dim[3] = {PR_HD, (cuuint64_t)r.n_kv * r.G, (cuuint64_t)n_tok};
    // (a dimension of one may come with any stride)
    const cuuint64_t stride[2] = {(cuuint64_t)(r.n_kv * r.G > 1 ? r.q_head : PR_HD) * 2,
                                  (cuuint64_t)(n_tok > 1 ? r.q_tok : PR_HD) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)r.G, (cuuint32_t)(TA_TILE / r.G)},
                     one[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(r.q), dim,
               stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// One warp per (token, head) of the tiles' tokens: parts joined, normalised, stored.  (A
// launch of its own: a warp that has eight parts' loads in flight and many warps to an SM;
// at the end of the few-row kernel's CTAs the same reads took 5 us of each.)
constexpr int TJ_WARPS = 8;
__global__ void __launch_bounds__(32 * TJ_WARPS) join_parts_kernel(const TileAttnParams p,
                                                                   int parts, int n_tok) {
    const int lane = threadIdx.x & 31, H = p.r.n_kv * p.r.G;
    const int64_t at = (int64_t)blockIdx.x * TJ_WARPS + (threadIdx.x >> 5);
    const int tok = (int)(at / H), h = (int)(at - (int64_t)tok * H);
    pdl_wait();
    if (tok >= n_tok || tok < p.bounds[0] || tok >= p.bounds[p.n_seg]) return;
    if (!p.prefix_lens) {
        int lo = 0, hi = p.n_seg - 1;               // the token's request
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.bounds[mid + 1] > tok) hi = mid; else lo = mid + 1;
        }
        int t0, n;
        segment(p, lo, t0, n);
        if (n == 0) return;                         // the few-row kernel's
    }
    const PartSum s = join_parts(p.parts_out, p.parts_ml, p.part_rows, parts, at, 4 * lane);
    const float inv = s.l != 0.f ? 1.f / s.l : 0.f;
    *reinterpret_cast<uint2*>(p.r.out + (int64_t)tok * p.r.o_tok + (int64_t)h * p.r.o_head +
                              4 * lane) =
        make_uint2(pack_bf16x2(s.o.x * inv, s.o.y * inv), pack_bf16x2(s.o.z * inv, s.o.w * inv));
    if (lane == 0 && p.r.lse)
        p.r.lse[(int64_t)tok * p.r.lse_tok + h] =
            s.l != 0.f ? (s.m + log2f(s.l)) * PR_LN2 : -INFINITY;
}

}  // namespace

int launch_tile_attn(const char* who, TileAttnParams p, int tiles, int max_tiles, int n_tok,
                     cudaStream_t s) {
    p.head_chunks = p.r.n_kv > 1 ? (int)(p.r.sh / 64) : 0;
    CUtensorMap mq = {}, mk, mv;
    CUresult cr = TA_TILE % p.r.G == 0 ? encode_q(&mq, p.r, n_tok) : CUDA_SUCCESS;
    if (cr == CUDA_SUCCESS)
        cr = encode_plane(&mk, p.r.k, p.r.n_kv, p.r.num_blocks, 64 * p.head_chunks, p.r.st, p.r.sb);
    if (cr == CUDA_SUCCESS)
        cr = encode_plane(&mv, p.r.v, p.r.n_kv, p.r.num_blocks, 64 * p.head_chunks, p.r.st,
                          p.r.sb);
    LOCKS_REQUIRE(cr == CUDA_SUCCESS, LOCKS_ERR_LAUNCH,
                  "%s: cuTensorMapEncodeTiled failed (%d)", who, (int)cr);
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    const int smem = (int)sizeof(TileSmem) + 1024;
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
        cudaFuncSetAttribute(tile_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem);
        attr_done[dev] = true;
    }
    const int64_t items = (int64_t)tiles * p.r.n_kv * p.parts;
    LOCKS_REQUIRE((int64_t)max_tiles * p.r.n_kv * p.parts < (1 << 30), LOCKS_ERR_SIZE,
                  "%s: too many query rows in one call", who);
    // (with a CTA for every tile that is expected, nobody has to count them first: what
    // there is beyond is looked for while those are computed)
    p.tile_bound = items <= sm_count() ? tiles : 0;
    p.tile_more = p.tile_bound ? max_tiles - tiles : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items < sm_count() ? items : sm_count()), 1, 1);
    cfg.blockDim = dim3(TA_THREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, tile_attn_kernel, mq, mk, mv, p);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(e));
    return check_launch(who);
}

int launch_join_parts(const char* who, const TileAttnParams& p, int parts, int n_tok,
                      cudaStream_t s) {
    const int64_t rows = (int64_t)n_tok * p.r.n_kv * p.r.G;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows + TJ_WARPS - 1) / TJ_WARPS), 1, 1);
    cfg.blockDim = dim3(32 * TJ_WARPS, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, join_parts_kernel, p, parts, n_tok);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(e));
    return check_launch(who);
}

}  // namespace locks
