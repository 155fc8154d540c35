// Paged attention of many query rows at a time on the 5th-generation tensor cores:
// the prompt (and long-chunk) half of the windowed attention, and the shared part of
// the shared-prefix decode.
//
// A "segment" is a run of query tokens that read one table row: a request's new
// tokens, or the single tokens of the requests that share a prefix.  Its rows
// (token, query head of the KV head) are packed, row = token * G + head, and cut
// into tiles of up to 256.  One CTA takes a tile of one KV head and walks the pages
// the tile can see -- first pages and recent ones as one list -- eight pages = 128
// keys at a time:
//
//   S [128 rows x 128 keys] = Q K^T       tcgen05.mma, Q and K in shared memory
//   P = exp2(scale (S - m)), l += sum P   a thread per row: its row of S comes from
//                                         tensor memory, P goes back there in bf16
//   O [128 rows x 128] += P V             tcgen05.mma, A = P from tensor memory
//
// Two such streams run against each other, so that one's softmax hides behind the
// other's products.  With more than 128 rows each stream has 128 of them and both
// walk every key tile; with fewer, both have the same rows and take the key tiles in
// turn (joined at the end through shared memory): a decode batch is then not half
// idle.
//
// Warps 0-3 and 4-7: softmax of stream 0 and 1 (thread = row = tensor-memory lane).
// Warp 8: one thread issues all products.  Warp 9: fetches pages through the table by
// tiled tensor-map copies (a page of a KV head is two boxes of 16 tokens x 64
// channels, 128-byte swizzle) into a ring of five 32 KiB tiles that K and V share.
// Tensor memory: S / P of the streams in columns 0 and 128, O in 256 and 384.
//
// The running maximum is only raised when it grows by more than 2^8 (O and l then
// get rescaled): P stays below 2^8 and no row of O is touched in most steps.  P is
// rounded to bf16 because V is (both operands of the product have one type), half a
// step each; m, l, S and O are fp32.
//
// Every wait is bounded (status word; later waits then return at once, copies in
// flight are waited for and tensor memory is freed).  No multicast.
#include "common.cuh"
#include "paged_rows.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace locks {
namespace {

constexpr int TA_THREADS = 320;
constexpr int TA_RING = 5;
constexpr int TA_TILE = 128;                       // keys of a tile, rows of a stream
constexpr int TA_PAGES = TA_TILE / PR_PAGE;
constexpr int TA_HALF = TA_TILE * 128;             // bytes: 128 rows x 64 channels
constexpr int TA_BYTES = 2 * TA_HALF;
constexpr int TA_BOX = PR_PAGE * 256;              // bytes of a page of one plane and head
constexpr int TM_S = 0, TM_O = 256, TM_COLS = 512;
constexpr float TA_RAISE = 8.f;

struct __align__(1024) TileSmem {
    uint8_t q[2][TA_BYTES];
    uint8_t ring[TA_RING][TA_BYTES];
    uint64_t full[TA_RING], empty[TA_RING], tail;
    uint64_t q_full, s_full[2], p_ready[2], o_full[2];
    uint32_t tmem_base;
    int dead;
    int scan[TA_THREADS / 32];
    int seg, seg_tile, seg_tiles;
    float xm[TA_TILE], xl[TA_TILE];
};
static_assert(sizeof(TileSmem) + 1024 <= 232448, "one CTA's shared memory");

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
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

// a wait that gives up once any wait of the CTA has
__device__ __forceinline__ void ta_wait(TileSmem& sm, uint64_t* bar, uint32_t parity,
                                        int* status) {
    if (mbar_try_wait(bar, parity)) return;
    for (int it = 0; it < (1 << 22); ++it) {
        if (mbar_try_wait(bar, parity)) return;
        if (it > 64) {
            __nanosleep(32);
            if (*reinterpret_cast<volatile int*>(&sm.dead)) return;
        }
    }
    *reinterpret_cast<volatile int*>(&sm.dead) = 1;
    if (status) atomicExch(status, LOCKS_ST_WAIT_TIMEOUT);
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

// segment s: first token and token count (0 where the few-row kernel serves it)
__device__ __forceinline__ void segment(const TileAttnParams& p, int s, int& t0, int& n) {
    t0 = p.bounds[s];
    n = p.bounds[s + 1] - t0;
    if (!p.prefix_lens && n * p.r.G <= p.min_rows) n = 0;
    n = max(n, 0);
}

// which segment tile `target` belongs to: a block-wide scan over the segments
__device__ __forceinline__ bool find_tile(TileSmem& sm, const TileAttnParams& p, int target) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sm.seg = -1;
    int before = 0;
    for (int s0 = 0; s0 < p.n_seg; s0 += TA_THREADS) {
        const int s = s0 + tid;
        int t0, n = 0;
        if (s < p.n_seg) segment(p, s, t0, n);
        const int mine = (n * p.r.G + 2 * TA_TILE - 1) / (2 * TA_TILE);
        int x = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == 31) sm.scan[warp] = x;
        __syncthreads();
        int mine_from = before + x - mine, total = before;
#pragma unroll
        for (int w = 0; w < TA_THREADS / 32; ++w) {
            if (w < warp) mine_from += sm.scan[w];
            total += sm.scan[w];
        }
        if (target >= mine_from && target < mine_from + mine) {
            sm.seg = s;
            sm.seg_tile = mine - 1 - (target - mine_from);      // longest rows first
        }
        before = total;
        if (before > target) break;
    }
    __syncthreads();
    return sm.seg >= 0;
}

__global__ void __launch_bounds__(TA_THREADS, 1)
tile_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const TileAttnParams p) {
    extern __shared__ uint8_t ta_raw[];
    TileSmem& sm = *reinterpret_cast<TileSmem*>(
        ta_raw + ((1024u - (smem_u32(ta_raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // uniform, and known to be
    const int kh = blockIdx.y, part = blockIdx.z, G = p.r.G;
    if (!find_tile(sm, p, blockIdx.x)) return;
    const int seg = sm.seg, row0 = sm.seg_tile * 2 * TA_TILE;
    int t0, n_tok;
    segment(p, seg, t0, n_tok);
    const int rows = n_tok * G, n_rows = min(rows - row0, 2 * TA_TILE);
    const bool by_rows = n_rows > TA_TILE;          // else both streams share the rows

    // ---- keys of the tile --------------------------------------------------------
    int key_end, written, base_pos = 0;             // written: keys behind it never were
    const int32_t* table;
    PageList list;
    if (p.prefix_lens) {
        const int whole = min(max(p.prefix_lens[seg], 0) / PR_PAGE, p.r.bt_width);
        written = key_end = whole * PR_PAGE;
        table = p.r.table + (int64_t)t0 * p.r.bt_stride;
        list = page_list(0, key_end - 1, INT32_MAX, 0, p.r.bt_width);
    } else {
        written = p.r.seq_lens[seg];
        base_pos = written - n_tok;
        table = p.r.table + (int64_t)seg * p.r.bt_stride;
        list = page_list(base_pos + row0 / G, base_pos + (row0 + n_rows - 1) / G,
                         p.r.window, p.r.sinks, p.r.bt_width);
        key_end = list.key_end;
    }
    const int all_tiles = (list.n + TA_PAGES - 1) / TA_PAGES;
    const int per = (all_tiles + p.parts - 1) / p.parts;
    const int j0 = min(part * per, all_tiles), n_tiles = min(j0 + per, all_tiles) - j0;

    // ---- setup -------------------------------------------------------------------
    if (tid == 0) {
        sm.dead = 0;
        for (int i = 0; i < TA_RING; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
        mbar_init(&sm.tail, 1);
        mbar_init(&sm.q_full, 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.s_full[i], 1);
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
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = sm.tmem_base;

    if (warp == 9) {
        // ---- pages: K and V tiles in the order the products take them ---------------
        int slot = 0, issued = 0;
        auto fetch = [&](int j, bool is_v) {
            if (issued >= TA_RING)
                ta_wait(sm, &sm.empty[slot], (uint32_t)((issued / TA_RING) - 1) & 1u, p.status);
            if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&sm.dead))) return;
            const int v = (j0 + j) * TA_PAGES + (lane & 7);
            int blk = p.r.num_blocks;               // outside the map: zeros
            bool partial = false;
            int page = 0;
            if (v < list.n) {
                page = list.page(v);
                blk = min(max(table[page], 0), p.r.num_blocks - 1);
                partial = is_v && (page + 1) * PR_PAGE > written;
            }
            const uint32_t cut = __ballot_sync(0xffffffffu, lane < 8 && partial);
            uint64_t* bar = cut ? &sm.tail : &sm.full[slot];
            if (lane == 0) mbar_expect_tx(bar, TA_BYTES);
            __syncwarp();
            if (lane < TA_PAGES)
                tma_load_page(&sm.ring[slot][lane * TA_BOX], is_v ? &map_v : &map_k,
                              kh * p.head_chunks, blk, bar);
            if (cut) {
                // the sequence ends inside a page: what the cache holds behind it may
                // be anything, and 0 x NaN is not 0
                ta_wait(sm, &sm.tail, 0, p.status);
                __syncwarp();
                const int s = __ffs(cut) - 1;
                const int from = max(written - __shfl_sync(0xffffffffu, page, s) * PR_PAGE, 0);
                for (int e = lane; e < (PR_PAGE - from) * 16; e += 32)
                    *reinterpret_cast<uint4*>(
                        &sm.ring[slot][s * TA_BOX + ((from + (e >> 4)) >> 3) * 2048 +
                                       ((e >> 3) & 1) * 1024 + ((from + (e >> 4)) & 7) * 128 +
                                       (e & 7) * 16]) = make_uint4(0, 0, 0, 0);
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
        // a wait ran out: nobody consumed the last copies; they must land all the same
        if (*reinterpret_cast<volatile int*>(&sm.dead))
            for (int i = max(issued - TA_RING, 0); i < issued; ++i)
                mbar_wait(&sm.full[i % TA_RING], (uint32_t)(i / TA_RING) & 1u, p.status);
    } else if (warp == 8) {
        // ---- products -------------------------------------------------------------
        if (n_tiles > 0) {
            constexpr uint32_t ID_S = tc_idesc(TA_TILE, false), ID_O = tc_idesc(PR_HD, true);
            const uint64_t desc_q = tc_desc(smem_u32(sm.q), 16, 1024),
                           desc_k = tc_desc(smem_u32(sm.ring), 16, 2048),
                           desc_v = tc_desc(smem_u32(sm.ring), 1024, 2048);
            int slot = 0, taken = 0;
            auto take = [&]() {                     // the next tile of the ring
                const int s = slot;
                ta_wait(sm, &sm.full[s], (uint32_t)(taken / TA_RING) & 1u, p.status);
                __syncwarp();
                slot = slot + 1 == TA_RING ? 0 : slot + 1;
                ++taken;
                return s;
            };
            auto scores = [&](int i, int s) {
                tc_after_sync();
                const uint64_t a = desc_q + (uint64_t)((by_rows ? i : 0) * (TA_BYTES >> 4));
                const uint64_t b = desc_k + (uint64_t)(s * (TA_BYTES >> 4));
                if (tc_elect()) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint64_t in_row = (ks & 3) * 32 >> 4, half = ks >> 2;
                        tc_mma_ss(tmem + TM_S + i * TA_TILE, a + in_row + half * (TA_HALF >> 4),
                                  b + in_row + half * (1024 >> 4), ID_S, ks ? 1u : 0u);
                    }
                    tc_commit(&sm.s_full[i]);
                }
                __syncwarp();
            };
            auto values = [&](int i, int s, int t) { // stream i's tile number t
                ta_wait(sm, &sm.p_ready[i], (uint32_t)t & 1u, p.status);
                __syncwarp();
                tc_after_sync();
                const uint64_t b = desc_v + (uint64_t)(s * (TA_BYTES >> 4));
                if (tc_elect()) {
#pragma unroll
                    for (int ks = 0; ks < TA_PAGES; ++ks)
                        tc_mma_ts(tmem + TM_O + i * PR_HD, tmem + TM_S + i * TA_TILE + ks * 8,
                                  b + (uint64_t)((ks * TA_BOX) >> 4), ID_O, (t | ks) ? 1u : 0u);
                    tc_commit(&sm.o_full[i]);
                }
                __syncwarp();
            };
            auto release = [&](int s) {
                if (tc_elect()) tc_commit(&sm.empty[s]);
                __syncwarp();
            };
            int k_slot = take();
            ta_wait(sm, &sm.q_full, 0, p.status);
            __syncwarp();
            scores(0, k_slot);
            if (by_rows) {
                scores(1, k_slot);
                release(k_slot);
                for (int j = 0; j < n_tiles; ++j) {
                    const int v_slot = take();
                    values(0, v_slot, j);
                    if (j + 1 < n_tiles) {
                        k_slot = take();
                        scores(0, k_slot);
                    }
                    values(1, v_slot, j);
                    release(v_slot);
                    if (j + 1 < n_tiles) {
                        scores(1, k_slot);
                        release(k_slot);
                    }
                }
            } else {
                release(k_slot);
                if (n_tiles > 1) {
                    k_slot = take();
                    scores(1, k_slot);
                    release(k_slot);
                }
                for (int j = 0; j < n_tiles; ++j) {
                    const int v_slot = take();
                    values(j & 1, v_slot, j >> 1);
                    release(v_slot);
                    if (j + 2 < n_tiles) {
                        k_slot = take();
                        scores(j & 1, k_slot);
                        release(k_slot);
                    }
                }
            }
        }
    } else if (warp < 8) {
        // ---- Q into the swizzled K-major layout, 16 lanes to a row -------------------
        {
            // (rows behind the last one are zeros; every copy is on its way before the
            // first is waited for)
            const int piece = tid & 15;
#pragma unroll 8
            for (int k = 0; k < (by_rows ? 16 : 8); ++k) {
                const int row = (tid >> 4) + 16 * k, at = row0 + min(row, n_rows - 1);
                const int tok = at / G;
                const __nv_bfloat16* src = p.r.q + (int64_t)(t0 + tok) * p.r.q_tok +
                                           (int64_t)(kh * G + at - tok * G) * p.r.q_head +
                                           8 * piece;
                cp_async16(smem_u32(&sm.q[row >> 7][(piece >> 3) * TA_HALF +
                                                    tc_swz(row & 127, (piece & 7) << 4)]),
                           src, row < n_rows ? 16 : 0);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full);
        }
        // ---- softmax: stream i, thread = row ---------------------------------------
        const int i = warp >> 2, q4 = warp & 3;
        const int local = (by_rows ? i * TA_TILE : 0) + q4 * 32 + lane;
        const int row = row0 + min(local, n_rows - 1);
        const int tok = row / G;
        const int pos = p.prefix_lens ? p.r.seq_lens[t0 + tok] - 1 : base_pos + tok;
        const int last_key = min(pos, key_end - 1);
        const int first_key = pos >= p.r.window ? pos - p.r.window + 1 : 0;
        const int sinks = p.r.sinks;
        // (row order is position order only for a request's own tokens)
        const int w_last = __reduce_min_sync(0xffffffffu, last_key);
        const int w_first = __reduce_max_sync(0xffffffffu, first_key);
        const uint32_t lane_base = tmem + ((uint32_t)(q4 * 32) << 16);
        const uint32_t ts = lane_base + TM_S + i * TA_TILE, to = lane_base + TM_O + i * PR_HD;
        const float sl2 = p.r.scale_log2;
        float m = -INFINITY, l = 0.f;
        int t = 0;                                  // tiles of this stream so far
        for (int j = by_rows ? 0 : i; j < n_tiles; j += by_rows ? 1 : 2, ++t) {
            ta_wait(sm, &sm.s_full[i], (uint32_t)t & 1u, p.status);
            __syncwarp();
            tc_after_sync();
            uint32_t sr[TA_TILE];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32(ts + 32 * c, sr + 32 * c);
            tc_wait_ld();
            float* s = reinterpret_cast<float*>(sr);
            const int v0 = (j0 + j) * TA_PAGES;
            {
                const int lo_key = list.page(v0) * PR_PAGE;
                const int hi_key = list.page(v0 + TA_PAGES - 1) * PR_PAGE + PR_PAGE - 1;
                const bool clear = v0 + TA_PAGES <= list.n && hi_key <= w_last &&
                                   (lo_key >= w_first || hi_key < sinks);
                if (!clear) {
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
                }
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < TA_TILE - 4; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
            const float tile_max =
                fmaxf(max3(max3(mx[0], mx[1], mx[2]), mx[3], s[TA_TILE - 4]),
                      max3(s[TA_TILE - 3], s[TA_TILE - 2], s[TA_TILE - 1]));
            if (t == 0) {
                m = tile_max;
            } else if (__any_sync(0xffffffffu, (tile_max - m) * sl2 > TA_RAISE)) {
                // (m -inf: nothing seen so far, O and l are 0 and stay it)
                const float up = fmaxf(m, tile_max);
                const float f = m == -INFINITY ? 0.f : pr_exp2((m - up) * sl2);
                m = up;
                l *= f;
                ta_wait(sm, &sm.o_full[i], (uint32_t)(t - 1) & 1u, p.status);
                __syncwarp();
                tc_after_sync();
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t o[16];
                    tc_ld16(to + 16 * c, o);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tc_st16(to + 16 * c, o);
                }
            }
            const float base = m == -INFINITY ? 0.f : m * sl2;
            const float2 k2 = make_float2(sl2, sl2), b2 = make_float2(-base, -base);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 x = fma2(make_float2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), k2, b2);
                    x.x = pr_exp2(x.x);
                    x.y = pr_exp2(x.y);
                    sum[e & 1] = add2(sum[e & 1], x);
                    pk[e] = pack_bf16x2(x.x, x.y);
                }
                tc_st16(ts + 16 * c, pk);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tc_wait_st();
            tc_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_ready[i]);
        }
        // ---- results ---------------------------------------------------------------
        if (t > 0) {
            ta_wait(sm, &sm.o_full[i], (uint32_t)(t - 1) & 1u, p.status);
            __syncwarp();
            tc_after_sync();
        }
        // streams that share the rows: stream 1 hands over (m, l, O), column by column
        // (lane = bank), stream 0 weighs both
        float w0 = 1.f, w1 = 0.f;
        float* xo = reinterpret_cast<float*>(sm.ring[0]);
        if (!by_rows) {
            const int at = q4 * 32 + lane;
            // (both streams' last products are done: the ring is idle)
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (i == 1) {
                sm.xm[at] = m;
                sm.xl[at] = l;
                if (t > 0)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tc_ld32(to + 32 * c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            xo[(32 * c + e) * TA_TILE + at] = __uint_as_float(o[e]);
                    }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (i == 0) {
                const float m1 = sm.xm[at], l1 = sm.xl[at];
                const float up = fmaxf(m, m1);
                w0 = l > 0.f ? pr_exp2((m - up) * sl2) : 0.f;
                w1 = l1 > 0.f ? pr_exp2((m1 - up) * sl2) : 0.f;
                l = w0 * l + w1 * l1;
                m = up;
            }
        }
        if ((by_rows || i == 0) && p.parts_out == nullptr) {
            const float inv = l > 0.f ? 1.f / l : 0.f;
            const int h = kh * G + row - tok * G;
            __nv_bfloat16* out = p.r.out + (int64_t)(t0 + tok) * p.r.o_tok + (int64_t)h * p.r.o_head;
            const bool second = w1 > 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                if (t > 0) {
                    tc_ld32(to + 32 * c, o);
                    tc_wait_ld();
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    float f[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        f[x] = l > 0.f && w0 > 0.f ? w0 * __uint_as_float(o[e + x]) : 0.f;
                        if (second)
                            f[x] += w1 * xo[(32 * c + e + x) * TA_TILE + q4 * 32 + lane];
                        f[x] *= inv;
                    }
                    if (local < n_rows)
                        *reinterpret_cast<uint4*>(out + 32 * c + e) =
                            make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                       pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
                }
            }
            if (p.r.lse && local < n_rows)
                p.r.lse[(int64_t)(t0 + tok) * p.r.lse_tok + h] =
                    l > 0.f ? (m * sl2 + log2f(l)) * PR_LN2 : -INFINITY;
        } else if (by_rows || i == 0) {
            // one of several parts: O relative to m, with (m in log2 units, l)
            const int h = kh * G + row - tok * G;
            const int64_t at = (int64_t)part * p.part_rows + (int64_t)(t0 + tok) * p.r.n_kv * G + h;
            float* out = p.parts_out + at * PR_HD;
            const bool second = w1 > 0.f;
            if (__any_sync(0xffffffffu, l > 0.f)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    if (t > 0) {
                        tc_ld32(to + 32 * c, o);
                        tc_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float f[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            f[x] = l > 0.f && w0 > 0.f ? w0 * __uint_as_float(o[e + x]) : 0.f;
                            if (second)
                                f[x] += w1 * xo[(32 * c + e + x) * TA_TILE + q4 * 32 + lane];
                        }
                        if (local < n_rows)
                            *reinterpret_cast<float4*>(out + 32 * c + e) =
                                make_float4(f[0], f[1], f[2], f[3]);
                    }
                }
            }
            if (local < n_rows)
                *reinterpret_cast<float2*>(p.parts_ml + 2 * at) =
                    make_float2(l > 0.f ? m * sl2 : -INFINITY, l);
        }
        tc_before_sync();
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

// One warp per (token, head) of the tiles' tokens: parts joined, normalised, stored.
constexpr int TJ_WARPS = 8;
__global__ void __launch_bounds__(32 * TJ_WARPS) join_parts_kernel(const TileAttnParams p,
                                                                   int n_tok) {
    const int lane = threadIdx.x & 31, H = p.r.n_kv * p.r.G;
    const int64_t at = (int64_t)blockIdx.x * TJ_WARPS + (threadIdx.x >> 5);
    const int tok = (int)(at / H), h = (int)(at - (int64_t)tok * H);
    if (tok >= n_tok || tok < p.bounds[0] || tok >= p.bounds[p.n_seg]) return;
    int lo = 0, hi = p.n_seg - 1;                   // the token's request
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.bounds[mid + 1] > tok) hi = mid; else lo = mid + 1;
    }
    if ((p.bounds[lo + 1] - p.bounds[lo]) * p.r.G <= p.min_rows) return;
    const PartSum s = join_parts(p.parts_out, p.parts_ml, p.part_rows, p.parts, at, 4 * lane);
    const float inv = s.l > 0.f ? 1.f / s.l : 0.f;
    *reinterpret_cast<uint2*>(p.r.out + (int64_t)tok * p.r.o_tok + (int64_t)h * p.r.o_head +
                              4 * lane) =
        make_uint2(pack_bf16x2(s.o.x * inv, s.o.y * inv), pack_bf16x2(s.o.z * inv, s.o.w * inv));
    if (lane == 0 && p.r.lse)
        p.r.lse[(int64_t)tok * p.r.lse_tok + h] =
            s.l > 0.f ? (s.m + log2f(s.l)) * PR_LN2 : -INFINITY;
}

}  // namespace

int launch_tile_attn(const char* who, TileAttnParams p, int max_tiles, cudaStream_t s) {
    p.head_chunks = p.r.n_kv > 1 ? (int)(p.r.sh / 64) : 0;
    CUtensorMap mk, mv;
    CUresult cr = encode_plane(&mk, p.r.k, p.r.n_kv, p.r.num_blocks, 64 * p.head_chunks, p.r.st, p.r.sb);
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
    tile_attn_kernel<<<dim3(max_tiles, p.r.n_kv, p.parts), TA_THREADS, smem, s>>>(mk, mv, p);
    return check_launch(who);
}

int launch_join_parts(const char* who, const TileAttnParams& p, int n_tok, cudaStream_t s) {
    const int64_t rows = (int64_t)n_tok * p.r.n_kv * p.r.G;
    join_parts_kernel<<<(unsigned)((rows + TJ_WARPS - 1) / TJ_WARPS), 32 * TJ_WARPS, 0, s>>>(
        p, n_tok);
    return check_launch(who);
}

}  // namespace locks
