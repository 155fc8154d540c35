// Paged attention of a few query rows per request with a sliding window and a few
// first tokens that stay visible.
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
// touched (a windowed cache has given them away).  A thread-block cluster owns
// (request, KV head): its warps take list entries in turn, each through its own
// ring of pages fetched with 16-byte cp.async, with an online softmax in fp32; the
// warps and then the CTAs join their (m, l, O) through shared memory, each CTA
// finishing a slice of the output.  No partials in HBM, one launch.
//
// P is split into two bf16 terms (P = hi + lo to 2^-17), so the product with V
// loses nothing to P's rounding; the second product costs tensor time that the
// memory-bound loop has to spare.  Keys that no row sees are filled with zeros
// on the way in, so what the cache holds there cannot reach the result.
#include <cooperative_groups.h>

#include "common.cuh"
#include "paged_rows.cuh"

namespace cg = cooperative_groups;

namespace locks {
namespace {

constexpr int RW = 8;                     // warps per CTA
constexpr int RTHREADS = RW * 32;
constexpr int RSTAGES = 2;
constexpr int ROW_PITCH = PR_HD * 2 + 16; // 272 B: conflict-free ldmatrix
constexpr int RACC_PITCH = PR_HD + 4;
constexpr int RMAX_CL = 16;

struct RowRing {
    uint8_t k[RSTAGES][PR_PAGE][ROW_PITCH];
    uint8_t v[RSTAGES][PR_PAGE][ROW_PITCH];
};
static_assert(sizeof(RowRing) >= 16 * RACC_PITCH * 4, "combine buffer must fit");

struct __align__(128) RowSmem {
    RowRing wb[RW];
    float cm[RW][16], cl[RW][16];
    float xm[RMAX_CL][16], xl[RMAX_CL][16];
    float xacc[16 * PR_HD + 16];
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

__global__ void __launch_bounds__(RTHREADS) row_attn_kernel(const RowAttnParams p) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    RowSmem& sm = *reinterpret_cast<RowSmem*>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int c = blockIdx.x, CL = gridDim.x, kh = blockIdx.y, r = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gid = lane >> 2, tig = lane & 3;
    const int G = p.G;
    // shared prefix: rows that belong to no group are left as they were
    int skip = 0;                             // whole prefix pages, attended already
    if (p.cu_groups) {
        if (r < p.cu_groups[0] || r >= p.cu_groups[p.n_groups]) return;
        int lo = 0, hi = p.n_groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_groups[mid + 1] > r) hi = mid; else lo = mid + 1;
        }
        skip = min(max(p.prefix_lens[lo], 0) / PR_PAGE, p.bt_width);
    }
    const int tok0 = p.cu_q ? p.cu_q[r] : r;
    const int n_q = p.cu_q ? p.cu_q[r + 1] - tok0 : 1;
    const int len = p.seq_lens[r];
    const int rows = n_q * G;
    if (rows > p.max_rows) return;            // the tiled kernel's
    const int32_t* table = p.table + (int64_t)r * p.bt_stride;

    // (the loop bound is the same for every CTA of the cluster)
    for (int rb = 0; rb * 16 < rows; ++rb) {
        const int row_a = rb * 16 + gid, row_b = row_a + 8;
        const int i_first = rb * 16 / G, i_last = min(rb * 16 + 15, rows - 1) / G;
        // rows behind the last one copy its position: never stored
        const int pos_a = len - n_q + min(row_a, rows - 1) / G;
        const int pos_b = len - n_q + min(row_b, rows - 1) / G;
        const PageList list = page_list(len - n_q + i_first, len - n_q + i_last, p.window,
                                        p.sinks, p.bt_width, skip);
        const int stride = RW * CL, first = c * RW + warp;
        const int n_mine = list.n > first ? (list.n - first + stride - 1) / stride : 0;

        // page and physical block of the warp's entries, 32 at a time
        int win_pg = 0, win_blk = 0, stage_pg[RSTAGES];
        auto load_window = [&](int it0) {
            const int it = it0 + lane;
            if (it < n_mine) {
                win_pg = list.page(first + it * stride);
                win_blk = min(max(table[win_pg], 0), p.num_blocks - 1);
            }
        };
        auto issue = [&](int it) {
            const int pg = __shfl_sync(0xffffffffu, win_pg, it & 31);
            const int blk = __shfl_sync(0xffffffffu, win_blk, it & 31);
            const int stage = it % RSTAGES, ch = lane & 15, h = lane >> 4;
            stage_pg[stage] = pg;
            const int64_t off = (int64_t)blk * p.sb + (int64_t)kh * p.sh + 8 * ch;
            const uint32_t kd = smem_u32(&sm.wb[warp].k[stage][0][16 * ch]);
            const uint32_t vd = smem_u32(&sm.wb[warp].v[stage][0][16 * ch]);
#pragma unroll
            for (int i = 0; i < PR_PAGE / 2; ++i) {
                const int t = h + 2 * i;
                const int nb = list.any_sees(pg * PR_PAGE + t) ? 16 : 0;
                const int64_t so = off + (int64_t)t * p.st;
                ra_cp16(kd + t * ROW_PITCH, p.k + so, nb);
                ra_cp16(vd + t * ROW_PITCH, p.v + so, nb);
            }
            ra_commit();
        };
        load_window(0);
        for (int it = 0; it < RSTAGES && it < n_mine; ++it) issue(it);

        uint32_t qa[8][4];
        {
            const int ia = row_a / G, ib = row_b / G;
            const bool live_a = row_a < rows, live_b = row_b < rows;
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
            const int stage = it % RSTAGES;
            const int key0 = stage_pg[stage] * PR_PAGE;
            if (it + 1 < n_mine) ra_wait<1>(); else ra_wait<0>();
            __syncwarp();
            const uint32_t kbase = smem_u32(&sm.wb[warp].k[stage]);
            const uint32_t vbase = smem_u32(&sm.wb[warp].v[stage]);
            float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const int t = (lane & 7) + 8 * ((lane >> 4) & 1);
                const uint32_t a0 = kbase + t * ROW_PITCH + 16 * ((lane >> 3) & 1);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    uint32_t kb[4];
                    ldmatrix_x4(kb, a0 + 32 * ks);
                    mma_bf16_k16(s0, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[0], kb[1]);
                    mma_bf16_k16(s1, qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kb[2], kb[3]);
                }
            }
            // scores in units of log2; x[0..3] row a, x[4..7] row b, keys 2 tig,
            // 2 tig + 1, 2 tig + 8, 2 tig + 9 of the page
            float x[8] = {s0[0], s0[1], s1[0], s1[1], s0[2], s0[3], s1[2], s1[3]};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = key0 + 2 * tig + (i & 1) + 8 * ((i >> 1) & 1);
                const int pos = i < 4 ? pos_a : pos_b;
                x[i] = list.sees(key, pos) ? x[i] * p.scale_log2 : -INFINITY;
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
            const float al_b = softmax4(x + 4, m_b, l_b);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                acc[i][0] *= al_a; acc[i][1] *= al_a;
                acc[i][2] *= al_b; acc[i][3] *= al_b;
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
                    mma_bf16_k16(acc[2 * dp], ph[0], ph[1], ph[2], ph[3], vb[0], vb[1]);
                    mma_bf16_k16(acc[2 * dp + 1], ph[0], ph[1], ph[2], ph[3], vb[2], vb[3]);
                    mma_bf16_k16(acc[2 * dp], pl[0], pl[1], pl[2], pl[3], vb[0], vb[1]);
                    mma_bf16_k16(acc[2 * dp + 1], pl[0], pl[1], pl[2], pl[3], vb[2], vb[3]);
                }
            }
            __syncwarp();                       // the stage is free
            if (it + RSTAGES < n_mine) {
                if (((it + RSTAGES) & 31) == 0) load_window(it + RSTAGES);
                issue(it + RSTAGES);
            }
        }

        // ---- the warps of the CTA -------------------------------------------------
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
        __syncthreads();                        // every ring is idle: fp32 scratch now
        float* wacc = reinterpret_cast<float*>(&sm.wb[warp]);
        if (tig == 0) {
            sm.cm[warp][gid] = m_a; sm.cl[warp][gid] = l_a;
            sm.cm[warp][gid + 8] = m_b; sm.cl[warp][gid + 8] = l_b;
        }
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
            *reinterpret_cast<float2*>(&wacc[gid * RACC_PITCH + 8 * nt + 2 * tig]) =
                make_float2(acc[nt][0], acc[nt][1]);
            *reinterpret_cast<float2*>(&wacc[(gid + 8) * RACC_PITCH + 8 * nt + 2 * tig]) =
                make_float2(acc[nt][2], acc[nt][3]);
        }
        __syncthreads();
        // ---- the CTAs of the cluster: CTA d finishes elements [d per_e, (d+1) per_e) --
        const int nr = min(16, rows - rb * 16), n_el = nr * PR_HD;
        const int per_e = (n_el + CL - 1) / CL;
        if (CL > 1) cluster.sync();             // peers run and are done with xacc
        for (int e = tid; e < n_el; e += RTHREADS) {
            const int row = e / PR_HD, d = e % PR_HD;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < RW; ++w) M = fmaxf(M, sm.cm[w][row]);
            float L = 0.f, o = 0.f;
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                const float lw = sm.cl[w][row];
                const float wt = lw > 0.f ? pr_exp2(sm.cm[w][row] - M) : 0.f;
                L += wt * lw;
                o += wt * reinterpret_cast<const float*>(&sm.wb[w])[row * RACC_PITCH + d];
            }
            const int dst = e / per_e;
            cluster.map_shared_rank(sm.xacc, dst)[c * per_e + (e - dst * per_e)] = o;
            if (d < CL) {
                cluster.map_shared_rank(&sm.xm[c][row], d)[0] = M;
                cluster.map_shared_rank(&sm.xl[c][row], d)[0] = L;
            }
        }
        if (CL > 1) cluster.sync();
        else __syncthreads();
        for (int e = c * per_e + tid; e < min((c + 1) * per_e, n_el); e += RTHREADS) {
            const int row = e / PR_HD, d = e % PR_HD;
            float M = -INFINITY;
            for (int cc = 0; cc < CL; ++cc) M = fmaxf(M, sm.xm[cc][row]);
            float L = 0.f, o = 0.f;
            for (int cc = 0; cc < CL; ++cc) {
                const float lc = sm.xl[cc][row];
                const float wt = lc > 0.f ? pr_exp2(sm.xm[cc][row] - M) : 0.f;
                L += wt * lc;
                o += wt * sm.xacc[cc * per_e + (e - c * per_e)];
            }
            const int at = rb * 16 + row, i = at / G, h = kh * G + at - i * G;
            if (p.parts) {
                // (one query token per request: i == 0, tok0 == r)
                const int64_t pr = (int64_t)tok0 * p.n_kv * G + h;
#pragma unroll 4
                for (int s = 0; s < p.parts; ++s) {
                    const int64_t x = s * p.part_rows + pr;
                    const float2 ml = *reinterpret_cast<const float2*>(p.parts_ml + 2 * x);
                    if (ml.y > 0.f) {
                        const float up = fmaxf(M, ml.x);
                        const float a = L > 0.f ? pr_exp2(M - up) : 0.f, b = pr_exp2(ml.x - up);
                        L = a * L + b * ml.y;
                        o = a * o + b * p.parts_o[x * PR_HD + d];
                        M = up;
                    }
                }
            }
            p.out[(int64_t)(tok0 + i) * p.o_tok + (int64_t)h * p.o_head + d] =
                __float2bfloat16_rn(L > 0.f ? o / L : 0.f);
            if (d == 0 && p.lse)
                p.lse[(int64_t)(tok0 + i) * p.lse_tok + h] =
                    L > 0.f ? (M + log2f(L)) * PR_LN2 : -INFINITY;
        }
        __syncthreads();
    }
    if (CL > 1) cluster.sync();                 // no CTA leaves while peers push to it
}

}  // namespace

int launch_row_attn(const char* who, const RowAttnParams& p, int n_req, cudaStream_t s) {
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    const int smem = (int)sizeof(RowSmem);
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
        cudaFuncSetAttribute(row_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem);
        attr_done[dev] = true;
    }
    int cl = 1;
    while (cl < 8 && cl * 2 * n_req * p.n_kv <= sm_count()) cl *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl, p.n_kv, n_req);
    cfg.blockDim = dim3(RTHREADS, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, row_attn_kernel, p);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(e));
    return check_launch(who);
}

}  // namespace locks
