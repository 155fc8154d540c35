// Step bookkeeping from request lengths, for any number of new tokens per
// request: where every new token goes in the paged cache, which blocks the step
// takes from the free list, and the lengths after it.
//
// With L_r tokens cached, n_r new ones, W table columns, F blocks in the free
// list of which `taken` are gone:
//   pages(x) = ceil(x / page)                    old_r = pages(L_r)
//   cu_r     = sum_{i<r} n_i                     (token layout of the step)
//   need_r   = pages(L_r + n_r) - old_r          if the request fits, else 0
//   upto_r   = sum_{i<=r} need_i
//   granted  = fits and (need_r == 0 or taken + upto_r <= F)
//   token i: pos = L_r + i, block = table[r, pos / page]            below old_r
//                                 = free[taken + upto_r - need_r + pos / page - old_r]
//            slot = block * page + pos % page     (-1 in a refused request)
// upto is monotone, so the granted takers are a prefix of the takers and the
// blocks they take are contiguous in the list: no atomics, same result every run.
//
// One launch.  Every CTA of the one cluster scans all requests itself (two block
// scans over at most 4096 of them), keeps (cu, length, first free index) in shared
// memory and fills its share of the tokens, each found by a binary search over cu.
// The outputs may be the inputs (lens_out = seq_lens, taken_out = taken): nothing
// is written before the cluster barrier behind the reads.  Bound by latency: the
// scan's two barriers and one table load; the large end writes 16 B a token.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace locks {
namespace {

constexpr int AP_FEW = 128, AP_MANY = 1024;      // threads of a CTA: small steps, large ones
constexpr int AP_MAX_REQS = 4096;
constexpr int AP_MAX_CL = 16;

struct PlanParams {
    const int32_t* seq_lens;
    const int32_t* n_new;
    int32_t* table;
    int64_t bt_stride;
    const int32_t* free_blocks;
    const int32_t* taken;
    int64_t* slot;
    int64_t* pos;
    int32_t* cu;
    int32_t* lens_out;
    int32_t* taken_out;
    int* status;
    int n_req, width, n_free, cap, page;
};

// exclusive prefix sum of one value per thread over the block; `total` on every
// thread.  Two barriers.
template <int THREADS>
__device__ __forceinline__ int block_excl_scan(int v, int* sh, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();                    // the previous use of sh is over
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const int s = sh[w];
        if (w < warp) before += s;
        total += s;
    }
    return before + x - v;
}

__device__ __forceinline__ int pages_of(int tokens, int page) {
    return (int)(((int64_t)tokens + page - 1) / page);
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) append_plan_kernel(const PlanParams p) {
    extern __shared__ int sh_dyn[];
    int* s_cu = sh_dyn;                          // n_req + 1
    int* s_len = s_cu + p.n_req + 1;             // n_req
    int* s_first = s_len + p.n_req;              // n_req: first free index, -1 refused
    __shared__ int sh[THREADS / 32];
    __shared__ int s_taken_max, s_refused;
    const int tid = threadIdx.x, rank = blockIdx.x, CL = gridDim.x;
    const int per = (p.n_req + THREADS - 1) / THREADS;
    const int r0 = min(tid * per, p.n_req), r1 = min(r0 + per, p.n_req);
    if (tid == 0) { s_taken_max = 0; s_refused = 0; }
    pdl_wait();                                  // (the lengths may be the last launch's)

    // ---- tokens -----------------------------------------------------------------
    int n = 0;
    for (int r = r0; r < r1; ++r) {
        s_len[r] = max(p.seq_lens[r], 0);
        s_cu[r] = max(p.n_new[r], 0);            // the count, for now
        n += s_cu[r];
    }
    int total;
    int run = block_excl_scan<THREADS>(n, sh, total);
    for (int r = r0; r < r1; ++r) {
        const int c = s_cu[r];
        s_cu[r] = run;
        run += c;
    }
    if (tid == 0) s_cu[p.n_req] = total;
    __syncthreads();
    // ---- blocks -----------------------------------------------------------------
    const int taken = max(*p.taken, 0);
    auto need_of = [&](int r, bool& fits) {
        const int len = s_len[r], c = s_cu[r + 1] - s_cu[r];
        const int64_t end = (int64_t)len + c;
        fits = end <= (int64_t)p.width * p.page && s_cu[r + 1] <= p.cap;
        return fits ? pages_of((int)end, p.page) - pages_of(len, p.page) : 0;
    };
    int need = 0;
    bool fits;
    for (int r = r0; r < r1; ++r) need += need_of(r, fits);
    int all_need;
    int upto = block_excl_scan<THREADS>(need, sh, all_need);
    int my_max = 0;
    bool refused = false;
    for (int r = r0; r < r1; ++r) {
        const int d = need_of(r, fits);
        upto += d;
        const bool ok = fits && (d == 0 || (int64_t)taken + upto <= p.n_free);
        s_first[r] = ok ? taken + upto - d : -1;
        refused |= !ok;
        if (ok && d) my_max = upto;
    }
    if (my_max) atomicMax(&s_taken_max, my_max);
    if (refused) s_refused = 1;
    if (CL > 1) cg::this_cluster().sync();       // every CTA has read the inputs
    else __syncthreads();

    // ---- outputs ----------------------------------------------------------------
    if (rank == 0) {
        for (int r = tid; r < p.n_req; r += THREADS) {
            p.cu[r] = s_cu[r];
            p.lens_out[r] = s_len[r] + (s_first[r] >= 0 ? s_cu[r + 1] - s_cu[r] : 0);
        }
        if (tid == 0) {
            p.cu[p.n_req] = total;
            *p.taken_out = taken + s_taken_max;
            if (s_refused && p.status) atomicExch(p.status, LOCKS_ST_PLAN_REFUSED);
        }
    }
    for (int t = rank * THREADS + tid; t < p.cap; t += CL * THREADS) {
        if (t >= total) { p.slot[t] = -1; p.pos[t] = 0; continue; }
        int lo = 0, hi = p.n_req - 1;            // the request with cu[r] <= t < cu[r+1]
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_cu[mid + 1] > t) hi = mid; else lo = mid + 1;
        }
        const int len = s_len[lo], pos = len + (t - s_cu[lo]), first = s_first[lo];
        p.pos[t] = pos;
        if (first < 0) { p.slot[t] = -1; continue; }
        const int pg = pos / p.page, in = pos - pg * p.page, fresh = pg - pages_of(len, p.page);
        int32_t* entry = p.table + (int64_t)lo * p.bt_stride + pg;
        const int blk = fresh >= 0 ? p.free_blocks[first + fresh] : *entry;
        if (fresh >= 0 && in == 0) *entry = blk;
        p.slot[t] = blk < 0 ? -1 : (int64_t)blk * p.page + in;
    }
}

}  // namespace
}  // namespace locks

using namespace locks;

extern "C" int locks_append_plan(const int32_t* seq_lens, const int32_t* n_new,
                                 int32_t* block_table, int64_t bt_stride, int bt_width,
                                 const int32_t* free_blocks, int n_free,
                                 const int32_t* taken, int64_t* slot_mapping,
                                 int64_t* positions, int32_t* cu_tokens,
                                 int32_t* lens_out, int32_t* taken_out, int n_req,
                                 int max_tokens, int page, int* status,
                                 locks_stream_t stream) {
    LOCKS_REQUIRE(seq_lens && n_new && block_table && taken && cu_tokens && lens_out &&
                      taken_out && (free_blocks || n_free == 0) &&
                      ((slot_mapping && positions) || max_tokens == 0),
                  LOCKS_ERR_ARG, "locks_append_plan: null pointer argument");
    LOCKS_REQUIRE(n_req >= 1 && bt_width >= 1 && bt_stride >= bt_width && n_free >= 0 &&
                      max_tokens >= 0 && page >= 1 &&
                      (int64_t)bt_width * page <= INT32_MAX,
                  LOCKS_ERR_ARG, "locks_append_plan: bad size argument");
    LOCKS_REQUIRE(n_req <= AP_MAX_REQS, LOCKS_ERR_SIZE,
                  "locks_append_plan: at most %d requests, got %d", AP_MAX_REQS, n_req);
    PlanParams p;
    p.seq_lens = seq_lens; p.n_new = n_new;
    p.table = block_table; p.bt_stride = bt_stride; p.width = bt_width;
    p.free_blocks = free_blocks; p.n_free = n_free; p.taken = taken;
    p.slot = slot_mapping; p.pos = positions; p.cu = cu_tokens;
    p.lens_out = lens_out; p.taken_out = taken_out;
    p.status = status; p.n_req = n_req; p.cap = max_tokens; p.page = page;
    // One small CTA while a thread has about two requests and two tokens at most.  Calls
    // in a graph, us, 128 threads against CTAs of 1024 (a wider scan, but a barrier of 32
    // warps), requests x tokens of the step: 1 x 1 2.9 and 4.7, 16 x 128 3.1 and 4.9,
    // 64 x 256 4.1 and 5.0, 256 x 256 4.8 and 5.2; on the other side 16 x 512 5.1 and 4.9,
    // 64 x 512 5.9 and 5.1, 256 x 512 7.0 and 5.4, 512 x 512 7.9 and 5.6, 1024 x 1024 14.7
    // and 6.7.  256 requests, 65536 tokens: 11 with 16 CTAs of 1024, 20 with 8 of 512.
    const bool few = n_req <= 2 * AP_FEW && max_tokens <= 2 * AP_FEW;
    void (*kernel)(const PlanParams) =
        few ? append_plan_kernel<AP_FEW> : append_plan_kernel<AP_MANY>;
    const int smem = (3 * n_req + 1) * (int)sizeof(int);
    static bool attr_done[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
        cudaFuncSetAttribute(append_plan_kernel<AP_MANY>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (3 * AP_MAX_REQS + 1) * (int)sizeof(int));
        cudaFuncSetAttribute(append_plan_kernel<AP_MANY>,
                             cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        attr_done[dev] = true;
    }
    int cl = 1;
    while (!few && cl < AP_MAX_CL && cl * AP_MANY < max_tokens) cl *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl, 1, 1);
    cfg.blockDim = dim3(few ? AP_FEW : AP_MANY, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "locks_append_plan: %s", cudaGetErrorString(e));
    pdl_break();             // the scorer reads block tables before its wait
    return check_launch("locks_append_plan");
}
