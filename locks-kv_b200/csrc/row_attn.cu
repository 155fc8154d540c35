// Paged attention of a few query rows per request with a sliding window and a few
// first tokens that stay visible; also the requests' own part of the shared-prefix
// decode.
//
//   query token i of a request with n_q new tokens and L cached ones (the new ones
//   among them) sits at position p = L - n_q + i and sees key j when
//       j <= p  and  (j > p - window  or  j < sinks)
//   out = softmax(scale q K^T) V over the seen keys; a row that sees none is 0 with
//   a log-sum-exp of -inf.
//
// The G query heads of a KV head and the query tokens share its keys: rows
// (token, head) are packed, 16 to a warp-level fragment, so a page is fetched once
// for all of them.  The pages a block of rows can see are two runs -- the first
// pages and the recent ones -- walked as one list; the pages between are never
// touched (a windowed cache has given them away).  Every warp takes list entries in
// turn through its own ring of pages fetched with 16-byte cp.async, with an online
// softmax in fp32; the warps join their (m, l, O) through shared memory.
//
// Bound by memory; what has to be hidden is latency, and there are two regimes:
//   many (request, KV head) pairs   one small CTA each, several to an SM, so that one's
//                                   start and end overlap the others' pages;
//   few                             a thread-block cluster each: its CTAs push (m, l, O)
//                                   into each other's shared memory and finish a slice
//                                   of the output each -- no partials in HBM, one launch;
//   few, very long lists            the small CTAs again, many to a pair, their results
//                                   joined by a launch behind them.
//
// P is split into two bf16 terms (P = hi + lo to 2^-17), so the product with V
// loses nothing to P's rounding; with up to 8 rows both terms share one product, above
// the second one costs tensor time that the memory-bound loop has to spare.  Keys that no
// row sees are filled with zeros on the way in, so what the cache holds there cannot reach
// the result.
//
// Behind the tiled kernel of the same call it is launched programmatically: it starts on
// SMs that have run out of tiles (the tiled kernel lets it once all of its CTAs run, when
// everything earlier on the stream is done) and waits for that kernel only before it ends.
#include <cooperative_groups.h>

#include "common.cuh"
#include "paged_rows.cuh"

namespace cg = cooperative_groups;

namespace locks {
namespace {

constexpr int ROW_PITCH = PR_HD * 2 + 16; // 272 B: conflict-free ldmatrix
constexpr int RACC_PITCH = PR_HD + 4;
constexpr int RMAX_CL = 16;

template <int STAGES>
struct RowRing {
    uint8_t k[STAGES][PR_PAGE][ROW_PITCH];
    uint8_t v[STAGES][PR_PAGE][ROW_PITCH];
};
static_assert(sizeof(RowRing<2>) >= 16 * RACC_PITCH * 4, "combine buffer must fit");

template <int WARPS, int STAGES, bool CLUSTER>
struct __align__(128) RowSmem {
    RowRing<STAGES> wb[WARPS];
    float cm[WARPS][16], cl[WARPS][16];
    // what the other CTAs of a cluster push here
    float xm[CLUSTER ? RMAX_CL : 1][16], xl[CLUSTER ? RMAX_CL : 1][16];
    float xacc[CLUSTER ? 16 * PR_HD + 16 * RMAX_CL : 1];
};

__device__ __forceinline__ void ra_cp16(uint32_t dst, const void* src, int src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void ra_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void ra_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void axpy4(float4& o, float w, const float4 v) {
    o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y);
    o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
}

// HI: rows are taken 16 to a block, else 8
template <int WARPS, int STAGES, bool CLUSTER, bool HI>
__global__ void __launch_bounds__(WARPS * 32) row_attn_kernel(const RowAttnParams p) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    using Smem = RowSmem<WARPS, STAGES, CLUSTER>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    constexpr int THREADS = WARPS * 32, BLOCK = HI ? 16 : 8;
    const int c = blockIdx.x, CL = gridDim.x;    // the pair's CTA, of how many
    const int kh = blockIdx.y, r = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gid = lane >> 2, tig = lane & 3;
    const int G = p.G;
    // first launch of its call: everything before it on the stream is done, and the next
    // launch may line up.  (Beside the tiled kernel that wait comes at the end.)
    if (!p.beside) {
        pdl_wait();
        pdl_trigger();
    }
    const int len = p.seq_lens[r];
    // shared prefix: the row's group, all bounds read at once; rows that belong to none
    // are left as they were
    int skip = 0;                             // whole prefix pages, attended already
    if (p.cu_groups) {
        int pre = -1;
        if (r >= p.cu_groups[0])
            for (int g0 = 0; g0 < p.n_groups; g0 += 32) {
                const int g = min(g0 + lane, p.n_groups - 1);
                const int end = p.cu_groups[g + 1], mine = max(p.prefix_lens[g], 0);
                const uint32_t in = __ballot_sync(0xffffffffu, end > r);
                if (in) { pre = __shfl_sync(0xffffffffu, mine, __ffs(in) - 1); break; }
            }
        if (pre < 0) {
            pdl_wait();
            return;
        }
        skip = min(pre / PR_PAGE, p.bt_width);
    }
    const int tok0 = p.cu_q ? p.cu_q[r] : r;
    const int n_q = p.cu_q ? p.cu_q[r + 1] - tok0 : 1;
    // (bounds that leave q are cut off; n_q still says where the request's queries sit)
    const int rows = tok0 < 0 ? 0 : min(n_q, p.n_tok - tok0) * G;
    if (rows > p.max_rows) {                  // the tiled kernel's
        pdl_wait();
        return;
    }
    const int32_t* table = p.table + (int64_t)r * p.bt_stride;

    // (the loop bound is the same for every CTA of the cluster)
    for (int rb = 0; rb * BLOCK < rows; ++rb) {
        const int row_a = rb * BLOCK + gid, row_b = row_a + 8;     // (row_b with HI only)
        const int i_first = rb * BLOCK / G, i_last = min(rb * BLOCK + BLOCK - 1, rows - 1) / G;
        // rows behind the last one copy its position: never stored
        const int pos_a = len - n_q + min(row_a, rows - 1) / G;
        const int pos_b = len - n_q + min(row_b, rows - 1) / G;
        const PageList list = page_list(len - n_q + i_first, len - n_q + i_last, p.window,
                                        p.sinks, p.bt_width, skip);
        const int stride = WARPS * CL, first = c * WARPS + warp;
        const int n_mine = list.n > first ? (list.n - first + stride - 1) / stride : 0;

        // the warp's entries, 32 at a time: page (bit 31: every row sees all of it) and
        // physical block
        int win_pg = 0, win_blk = 0, stage_pg[STAGES];
        auto load_window = [&](int it0) {
            const int it = it0 + lane;
            if (it < n_mine) {
                const int pg = list.page(first + it * stride);
                win_blk = min(max(table[pg], 0), p.num_blocks - 1);
                win_pg = pg | (list.all_see(pg) ? (int)0x80000000 : 0);
            }
        };
        auto issue = [&](int it) {
            const int pg = __shfl_sync(0xffffffffu, win_pg, it & 31);
            const int blk = __shfl_sync(0xffffffffu, win_blk, it & 31);
            const int stage = it % STAGES, ch = lane & 15, h = lane >> 4;
            stage_pg[stage] = pg;
            const int64_t off = (int64_t)blk * p.sb + (int64_t)kh * p.sh + 8 * ch + h * p.st;
            const __nv_bfloat16 *ks = p.k + off, *vs = p.v + off;
            const uint32_t kd = smem_u32(&sm.wb[warp].k[stage][h][16 * ch]);
            const uint32_t vd = smem_u32(&sm.wb[warp].v[stage][h][16 * ch]);
            if (pg < 0) {
#pragma unroll
                for (int i = 0; i < PR_PAGE / 2; ++i) {
                    ra_cp16(kd + 2 * i * ROW_PITCH, ks + 2 * i * p.st, 16);
                    ra_cp16(vd + 2 * i * ROW_PITCH, vs + 2 * i * p.st, 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < PR_PAGE / 2; ++i) {
                    const int nb = list.any_sees(pg * PR_PAGE + h + 2 * i) ? 16 : 0;
                    ra_cp16(kd + 2 * i * ROW_PITCH, ks + 2 * i * p.st, nb);
                    ra_cp16(vd + 2 * i * ROW_PITCH, vs + 2 * i * p.st, nb);
                }
            }
            ra_commit();
        };
        load_window(0);
#pragma unroll
        for (int it = 0; it < STAGES - 1; ++it) {
            if (it < n_mine) issue(it);
            else ra_commit();                   // (an empty group: the counts below hold)
        }

        uint32_t qa[8][4];
        {
            const int ia = row_a / G, ib = row_b / G;
            const bool live_a = row_a < rows, live_b = HI && row_b < rows;
            const uint32_t* ra = reinterpret_cast<const uint32_t*>(
                p.q + (int64_t)(tok0 + ia) * p.q_tok + (int64_t)(kh * G + row_a - ia * G) * p.q_head);
            const uint32_t* rbp = reinterpret_cast<const uint32_t*>(
                p.q + (int64_t)(tok0 + ib) * p.q_tok + (int64_t)(kh * G + row_b - ib * G) * p.q_head);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                qa[ks][0] = live_a ? ra[8 * ks + tig] : 0u;
                qa[ks][1] = live_b ? rbp[8 * ks + tig] : 0u;
                qa[ks][2] = live_a ? ra[8 * ks + 4 + tig] : 0u;
                qa[ks][3] = live_b ? rbp[8 * ks + 4 + tig] : 0u;
            }
        }
        float acc[16][4];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;

        for (int it = 0; it < n_mine; ++it) {
            // the stage of the page before last's products is free: refill it first
            if (it + STAGES - 1 < n_mine) {
                if (((it + STAGES - 1) & 31) == 0) load_window(it + STAGES - 1);
                issue(it + STAGES - 1);
            } else {
                ra_commit();
            }
            const int stage = it % STAGES;
            ra_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t kbase = smem_u32(&sm.wb[warp].k[stage]);
            const uint32_t vbase = smem_u32(&sm.wb[warp].v[stage]);
            // (two chains of products per half page: each is latency, not work)
            float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
            float u0[4] = {0.f, 0.f, 0.f, 0.f}, u1[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const int t = (lane & 7) + 8 * ((lane >> 4) & 1);
                const uint32_t a0 = kbase + t * ROW_PITCH + 16 * ((lane >> 3) & 1);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    uint32_t kb[4];
                    ldmatrix_x4(kb, a0 + 32 * ks);
                    mma_bf16_k16(ks & 1 ? u0 : s0, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3],
                                 kb[0], kb[1]);
                    mma_bf16_k16(ks & 1 ? u1 : s1, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3],
                                 kb[2], kb[3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) { s0[i] += u0[i]; s1[i] += u1[i]; }
            }
            // scores in units of log2; x[0..3] row a, x[4..7] row b, keys 2 tig,
            // 2 tig + 1, 2 tig + 8, 2 tig + 9 of the page
            float x[8] = {s0[0], s0[1], s1[0], s1[1], s0[2], s0[3], s1[2], s1[3]};
            const int pg = stage_pg[stage];
#pragma unroll
            for (int i = 0; i < (HI ? 8 : 4); ++i) x[i] *= p.scale_log2;
            if (pg >= 0) {
#pragma unroll
                for (int i = 0; i < (HI ? 8 : 4); ++i) {
                    const int key = pg * PR_PAGE + 2 * tig + (i & 1) + 8 * ((i >> 1) & 1);
                    if (!list.sees(key, i < 4 ? pos_a : pos_b)) x[i] = -INFINITY;
                }
            }
            auto softmax4 = [&](float* xs, float& m, float& l) {
                float mx = fmaxf(fmaxf(xs[0], xs[1]), fmaxf(xs[2], xs[3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m, mx);
                const float base = mn == -INFINITY ? 0.f : mn;   // nothing seen yet
                const float alpha = pr_exp2(m - base);
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) { xs[i] = pr_exp2(xs[i] - base); s += xs[i]; }
                l = l * alpha + s;
                m = mn;
                return alpha;
            };
            const float al_a = softmax4(x, m_a, l_a);
            float al_b = 1.f;
            if (HI) al_b = softmax4(x + 4, m_b, l_b);
            else x[4] = x[5] = x[6] = x[7] = 0.f;
            if (!HI) al_b = al_a;
            // (the maximum of most pages is not a new one)
            if (__any_sync(0xffffffffu, al_a != 1.f || al_b != 1.f)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc[i][0] *= al_a; acc[i][1] *= al_a;
                    acc[i][2] *= al_b; acc[i][3] *= al_b;
                }
            }
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {       // (a, t0-7), (b, t0-7), (a, t8-15), (b, t8-15)
                const int o = (i & 1) * 4 + (i >> 1) * 2;
                ph[i] = pack_bf16x2(x[o], x[o + 1]);
                pl[i] = pack_bf16x2(x[o] - __uint_as_float(ph[i] << 16),
                                    x[o + 1] - __uint_as_float(ph[i] & 0xFFFF0000u));
            }
            {
                const int t = (lane & 7) + 8 * ((lane >> 3) & 1);
                const uint32_t a0 = vbase + t * ROW_PITCH + 16 * ((lane >> 4) & 1);
#pragma unroll
                for (int dp = 0; dp < 8; ++dp) {
                    uint32_t vb[4];
                    ldmatrix_x4_trans(vb, a0 + 32 * dp);
                    if (HI) {
                        mma_bf16_k16(acc[2 * dp], ph[0], ph[1], ph[2], ph[3], vb[0], vb[1]);
                        mma_bf16_k16(acc[2 * dp + 1], ph[0], ph[1], ph[2], ph[3], vb[2], vb[3]);
                        mma_bf16_k16(acc[2 * dp], pl[0], pl[1], pl[2], pl[3], vb[0], vb[1]);
                        mma_bf16_k16(acc[2 * dp + 1], pl[0], pl[1], pl[2], pl[3], vb[2], vb[3]);
                    } else {
                        // up to 8 rows: the lower terms ride in fragment rows 8-15
                        mma_bf16_k16(acc[2 * dp], ph[0], pl[0], ph[2], pl[2], vb[0], vb[1]);
                        mma_bf16_k16(acc[2 * dp + 1], ph[0], pl[0], ph[2], pl[2], vb[2], vb[3]);
                    }
                }
            }
            __syncwarp();                       // the stage is free
        }

        if (!HI)
#pragma unroll
            for (int i = 0; i < 16; ++i) { acc[i][0] += acc[i][2]; acc[i][1] += acc[i][3]; }
        // ---- the warps of the CTA -------------------------------------------------
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        if (HI) {
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
        }
        ra_wait<0>();
        float* wacc = reinterpret_cast<float*>(&sm.wb[warp]);     // the warp's idle ring
        if (tig == 0) {
            sm.cm[warp][gid] = m_a; sm.cl[warp][gid] = l_a;
            sm.cm[warp][gid + 8] = m_b; sm.cl[warp][gid + 8] = l_b;
        }
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
            *reinterpret_cast<float2*>(&wacc[gid * RACC_PITCH + 8 * nt + 2 * tig]) =
                make_float2(acc[nt][0], acc[nt][1]);
            if (HI)
                *reinterpret_cast<float2*>(&wacc[(gid + 8) * RACC_PITCH + 8 * nt + 2 * tig]) =
                    make_float2(acc[nt][2], acc[nt][3]);
        }
        const int nr = min(BLOCK, rows - rb * BLOCK), n_el = nr * (PR_HD / 4);
        if (CLUSTER) cg::this_cluster().sync(); // peers run, and are done with xacc
        else __syncthreads();
        // four channels of a row: (m, l, O) over the CTA's warps
        auto warps_sum = [&](int row, int d, float& M, float& L) {
            M = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm.cm[w][row]);
            L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float lw = sm.cl[w][row];
                const float wt = lw != 0.f ? pr_exp2(sm.cm[w][row] - M) : 0.f;
                L += wt * lw;
                axpy4(o, wt, *reinterpret_cast<const float4*>(
                                 reinterpret_cast<const float*>(&sm.wb[w]) + row * RACC_PITCH + d));
            }
            return o;
        };
        auto finish = [&](int row, int d, float M, float L, float4 o) {
            const int at = rb * BLOCK + row, i = at / G, h = kh * G + at - i * G;
            if (p.parts_o) {
                // one of several parts
                const int64_t x = (p.part + (CLUSTER ? 0 : c)) * p.part_rows +
                                  (int64_t)(tok0 + i) * p.n_kv * G + h;
                *reinterpret_cast<float4*>(p.parts_o + x * PR_HD + d) = o;
                if (d == 0)
                    *reinterpret_cast<float2*>(p.parts_ml + 2 * x) = make_float2(M, L);
                return;
            }
            // (a sum that is NaN makes the row NaN: only 0 is a row that saw nothing)
            const float inv = L != 0.f ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(p.out + (int64_t)(tok0 + i) * p.o_tok +
                                      (int64_t)h * p.o_head + d) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
            if (d == 0 && p.lse)
                p.lse[(int64_t)(tok0 + i) * p.lse_tok + h] =
                    L != 0.f ? (M + log2f(L)) * PR_LN2 : -INFINITY;
        };
        if (!CLUSTER) {
            for (int e = tid; e < n_el; e += THREADS) {
                float M, L;
                const int row = e / (PR_HD / 4), d = 4 * (e % (PR_HD / 4));
                const float4 o = warps_sum(row, d, M, L);
                finish(row, d, M, L, o);
            }
            if ((rb + 1) * BLOCK < rows) __syncthreads();       // the rings are idle again
        } else {
            // CTA k finishes the four-channel pieces [k per, (k + 1) per)
            cg::cluster_group cluster = cg::this_cluster();
            const int per = (n_el + CL - 1) / CL;
            for (int e = tid; e < n_el; e += THREADS) {
                float M, L;
                const int row = e / (PR_HD / 4), piece = e % (PR_HD / 4);
                const float4 o = warps_sum(row, 4 * piece, M, L);
                const int dst = e / per;
                *reinterpret_cast<float4*>(cluster.map_shared_rank(sm.xacc, dst) +
                                           4 * (c * per + e - dst * per)) = o;
                if (piece < CL) {
                    cluster.map_shared_rank(&sm.xm[c][row], piece)[0] = M;
                    cluster.map_shared_rank(&sm.xl[c][row], piece)[0] = L;
                }
            }
            cluster.sync();
            for (int e = c * per + tid; e < min((c + 1) * per, n_el); e += THREADS) {
                const int row = e / (PR_HD / 4);
                float M = -INFINITY, L = 0.f;
                for (int k = 0; k < CL; ++k) M = fmaxf(M, sm.xm[k][row]);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int k = 0; k < CL; ++k) {
                    const float lk = sm.xl[k][row];
                    const float wt = lk != 0.f ? pr_exp2(sm.xm[k][row] - M) : 0.f;
                    L += wt * lk;
                    axpy4(o, wt, *reinterpret_cast<const float4*>(
                                     &sm.xacc[4 * (k * per + e - c * per)]));
                }
                finish(row, 4 * (e % (PR_HD / 4)), M, L, o);
            }
            // (the next block's barrier keeps xacc; nobody pushes behind the last one)
        }
    }
    // launched beside the tiled kernel: the call is over when both are
    pdl_wait();
}

template <int WARPS, int STAGES, bool CLUSTER, bool HI>
int launch_row(const char* who, const RowAttnParams& p, int n_req, int splits,
               cudaStream_t s) {
    auto kernel = row_attn_kernel<WARPS, STAGES, CLUSTER, HI>;
    // clusters of 2, 4, 8 and 16 CTAs the device holds at once (a cluster lives in one
    // GPC, so that fewer of the large ones fit than SMs would suggest)
    static int fit[64][4] = {};
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    const int smem = (int)sizeof(RowSmem<WARPS, STAGES, CLUSTER>);
    const bool known = dev >= 0 && dev < 64;
    if (known && !attr_done[dev]) {
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (CLUSTER) {
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            for (int i = 0; i < 4; ++i)
                fit[dev][i] = max_active_clusters(kernel, 2 << i, WARPS * 32, smem);
        }
        attr_done[dev] = true;
    }
    int cl = splits;
    if (CLUSTER) {
        // the largest that lets every pair's cluster run at once
        cl = 2;
        for (int i = 1; i < 4; ++i)
            if (known && (int64_t)n_req * p.n_kv <= fit[dev][i]) cl = 2 << i;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl, p.n_kv, n_req);
    cfg.blockDim = dim3(WARPS * 32, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (CLUSTER) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cl;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(e));
    return check_launch(who);
}

}  // namespace

int launch_row_attn(const char* who, const RowAttnParams& p, int n_req, int most_rows,
                    int splits, cudaStream_t s) {
    // Small CTAs (four warps, three stages, two CTAs to an SM) once there are enough pairs
    // for most SMs; clusters of eight-warp CTAs below.  64 requests x 8 heads x 129 pages:
    // 87 us (6.2 TB/s); with two stages and three CTAs to an SM 120, with two warps 102,
    // with eight-warp CTAs, one to an SM, 125.  8 pairs x 257 pages in clusters of eight:
    // 9.6 us, with four-warp CTAs 10.5.
    const int64_t pairs = (int64_t)n_req * p.n_kv;
    const bool hi = most_rows > 8;
    if (2 * pairs > sm_count() || splits > 1)
        return hi ? launch_row<4, 3, false, true>(who, p, n_req, splits, s)
                  : launch_row<4, 3, false, false>(who, p, n_req, splits, s);
    return hi ? launch_row<8, 3, true, true>(who, p, n_req, 1, s)
              : launch_row<8, 3, true, false>(who, p, n_req, 1, s);
}

}  // namespace locks
