// Per-head RMS norm of the step's queries and keys, position rotation, and the
// K / V store into the paged cache, in one pass over the projection's output.
//
//   y = x / sqrt(mean_d x_d^2 + eps) * w_d         (skipped where w is null)
//   (y_i, y_j) <- (y_i c - y_j s, y_j c + y_i s)   for each rotated channel pair:
//                 j = i + rot/2 (half-split) or j = i + 1, i even (interleaved)
//   q row -> q_out, k row -> K cache at the token's slot, v row -> V cache
// All of it in fp32 with one rounding to bf16 at the end.
//
// Bound by memory: a row is read and written once, 2 * 256 B.  A half-warp owns a
// row (16 lanes x 8 channels = one 16-byte access per lane), so the norm is four
// shuffles and the half-split partner sits half/8 lanes away.  A warp takes NR_ROWS
// pairs of neighbouring rows of one token: their loads are all in flight before the
// first is used, and the token's slot, position and (cos | sin) row are read once.
#include "common.cuh"

namespace locks {
namespace {

constexpr int NR_HD = 128;
constexpr int NR_THREADS = 256;
constexpr int NR_HALVES = NR_THREADS / 16;
constexpr int NR_ROWS = 4;

enum RopeMode { ROPE_NONE, ROPE_PAIRS, ROPE_HALVES, ROPE_ANY };

struct NormRopeParams {
    const __nv_bfloat16 *q, *k, *v;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
    __nv_bfloat16* q_out;
    int64_t o_tok, o_head;
    __nv_bfloat16 *k_cache, *v_cache;
    int64_t cb, ct, ch;
    const int64_t *slot, *pos;
    const void* cos_sin;
    int64_t cs_row;
    const void *q_weight, *k_weight;
    int weight_f32, rot, neox, n_pos, num_blocks;
    int n_tok, H, n_kv, chunks;                    // chunks of 2 NR_ROWS heads a token
    float eps;
};

__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                      pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
// N consecutive table or weight values as fp32 (N a multiple of 4, 8-byte aligned
// for bf16 and 16-byte for fp32)
template <int N>
__device__ __forceinline__ void load_vals(const float* p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
        f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
    }
}
template <int N>
__device__ __forceinline__ void load_vals(const __nv_bfloat16* p, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p) + i);
        f[4 * i] = __uint_as_float(v.x << 16);
        f[4 * i + 1] = __uint_as_float(v.x & 0xFFFF0000u);
        f[4 * i + 2] = __uint_as_float(v.y << 16);
        f[4 * i + 3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <int MODE, class Tab>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const NormRopeParams p) {
    __shared__ float stage[MODE == ROPE_ANY ? NR_HALVES : 1][MODE == ROPE_ANY ? NR_HD : 1];
    const int half_id = threadIdx.x >> 4, lane = threadIdx.x & 15, side = half_id & 1;
    const int heads = p.H + 2 * p.n_kv;
    const int unit = blockIdx.x * (NR_THREADS / 32) + (threadIdx.x >> 5);
    const int t = unit / p.chunks;
    if (t >= p.n_tok) return;                    // (a whole warp)
    const int h0 = (unit - t * p.chunks) * (2 * NR_ROWS) + side;

    uint4 x[NR_ROWS];
#pragma unroll
    for (int i = 0; i < NR_ROWS; ++i) {
        const int h = h0 + 2 * i;
        x[i] = make_uint4(0, 0, 0, 0);
        if (h >= heads) continue;
        const __nv_bfloat16* src =
            h < p.H ? p.q + t * p.q_tok + h * p.q_head
            : h < p.H + p.n_kv ? p.k + t * p.k_tok + (h - p.H) * p.k_head
                               : p.v + t * p.v_tok + (h - p.H - p.n_kv) * p.v_head;
        x[i] = *reinterpret_cast<const uint4*>(src + 8 * lane);
    }
    const int64_t slot = p.slot[t];
    // the token's table row, as far as this lane's channels need it
    const int half = p.rot >> 1;
    const Tab* cs = static_cast<const Tab*>(p.cos_sin);
    const bool turns = 8 * lane < p.rot;
    const int hl = half >> 3;                    // half-split: lanes of one half
    const bool low = lane < hl;
    float c[8], s[8];
    if constexpr (MODE != ROPE_NONE) {
        cs += min(max(p.pos[t], (int64_t)0), (int64_t)p.n_pos - 1) * p.cs_row;
        if (MODE == ROPE_PAIRS && turns) {       // rot a multiple of 8
            float (&c4)[4] = reinterpret_cast<float (&)[4]>(c);
            float (&s4)[4] = reinterpret_cast<float (&)[4]>(s);
            load_vals(cs + 4 * lane, c4);
            load_vals(cs + half + 4 * lane, s4);
        }
        if (MODE == ROPE_HALVES && turns) {      // half a multiple of 8
            const int d = 8 * (low ? lane : lane - hl);
            load_vals(cs + d, c);
            load_vals(cs + half + d, s);
        }
    }
    const bool stored = slot >= 0 && (slot >> 4) < p.num_blocks;
    const int64_t at = stored ? (slot >> 4) * p.cb + (slot & 15) * p.ct : 0;
#pragma unroll
    for (int i = 0; i < NR_ROWS; ++i) {
        // (both half-warps of a warp run every round: the shuffles need all lanes)
        const int h = h0 + 2 * i;
        const bool is_q = h < p.H, is_k = !is_q && h < p.H + p.n_kv;
        uint4 y = x[i];
        float f[8];
        unpack8(x[i], f);
        const void* wt = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        if (wt) {
            const float rs = rsqrtf(ss * (1.f / NR_HD) + p.eps);
            float w[8];
            if (p.weight_f32) load_vals(static_cast<const float*>(wt) + 8 * lane, w);
            else load_vals(static_cast<const __nv_bfloat16*>(wt) + 8 * lane, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = f[e] * rs * w[e];
        }
        if constexpr (MODE == ROPE_PAIRS) {
            if (turns) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = f[2 * e], b = f[2 * e + 1];
                    f[2 * e] = a * c[e] - b * s[e];
                    f[2 * e + 1] = b * c[e] + a * s[e];
                }
            }
        } else if constexpr (MODE == ROPE_HALVES) {
            const int partner = turns ? (low ? lane + hl : lane - hl) : lane;
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __shfl_sync(0xffffffffu, f[e], partner, 16);
            if (turns) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    f[e] = low ? f[e] * c[e] - o[e] * s[e] : f[e] * c[e] + o[e] * s[e];
            }
        } else if constexpr (MODE == ROPE_ANY) {            // any even rot, any alignment
#pragma unroll
            for (int e = 0; e < 8; ++e) stage[half_id][8 * lane + e] = f[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = 8 * lane + e;
                if ((is_q || is_k) && d < p.rot) {
                    const bool first = p.neox ? d < half : (d & 1) == 0;
                    const int o = p.neox ? (first ? d + half : d - half) : d ^ 1;
                    const int j = p.neox ? (first ? d : d - half) : d >> 1;
                    const float cj = to_f32(cs[j]), sj = to_f32(cs[half + j]);
                    f[e] = first ? f[e] * cj - stage[half_id][o] * sj
                                 : f[e] * cj + stage[half_id][o] * sj;
                }
            }
            __syncwarp();
        }
        if (is_q || is_k) y = pack8(f);
        if (is_q) {
            *reinterpret_cast<uint4*>(p.q_out + t * p.o_tok + h * p.o_head + 8 * lane) = y;
        } else if (h < heads && stored) {
            const int kh = is_k ? h - p.H : h - p.H - p.n_kv;
            *reinterpret_cast<uint4*>((is_k ? p.k_cache : p.v_cache) + at + kh * p.ch +
                                      8 * lane) = y;
        }
    }
}

template <class Tab>
void launch_norm_rope(int mode, dim3 grid, cudaStream_t s, const NormRopeParams& p) {
    switch (mode) {
        case ROPE_NONE:   norm_rope_kernel<ROPE_NONE, Tab><<<grid, NR_THREADS, 0, s>>>(p); break;
        case ROPE_PAIRS:  norm_rope_kernel<ROPE_PAIRS, Tab><<<grid, NR_THREADS, 0, s>>>(p); break;
        case ROPE_HALVES: norm_rope_kernel<ROPE_HALVES, Tab><<<grid, NR_THREADS, 0, s>>>(p); break;
        default:          norm_rope_kernel<ROPE_ANY, Tab><<<grid, NR_THREADS, 0, s>>>(p); break;
    }
}

bool rows16(const void* p, int64_t a, int64_t b) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a % 8 == 0 && b % 8 == 0;
}

}  // namespace
}  // namespace locks

using namespace locks;

extern "C" int locks_norm_rope_write(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* key,
    int64_t k_stride_tok, int64_t k_stride_head, const void* val, int64_t v_stride_tok,
    int64_t v_stride_head, void* q_out, int64_t o_stride_tok, int64_t o_stride_head,
    void* k_cache, void* v_cache, int64_t kv_stride_block, int64_t kv_stride_tok,
    int64_t kv_stride_head, const int64_t* slot_mapping, const int64_t* positions,
    const void* cos_sin, int64_t cos_sin_row_stride, int n_positions, int rot_dim,
    int neox, int table_f32, const void* q_weight, const void* k_weight, int weight_f32,
    float eps, int n_tok, int n_heads, int n_kv, int head_dim, int page, int num_blocks,
    locks_stream_t stream) {
    LOCKS_REQUIRE(q && key && val && q_out && k_cache && v_cache && slot_mapping,
                  LOCKS_ERR_ARG, "locks_norm_rope_write: null pointer argument");
    LOCKS_REQUIRE(head_dim == NR_HD && page == 16, LOCKS_ERR_GEOMETRY,
                  "locks_norm_rope_write: supports head_dim 128 / page 16, got %d / %d",
                  head_dim, page);
    LOCKS_REQUIRE(n_tok >= 0 && n_heads >= 1 && n_kv >= 1 && num_blocks >= 1 &&
                      (int64_t)n_tok * (n_heads + 2 * n_kv) < (int64_t)1 << 31,
                  LOCKS_ERR_ARG, "locks_norm_rope_write: bad size argument");
    LOCKS_REQUIRE(rows16(q, q_stride_tok, q_stride_head) &&
                      rows16(key, k_stride_tok, k_stride_head) &&
                      rows16(val, v_stride_tok, v_stride_head) &&
                      rows16(q_out, o_stride_tok, o_stride_head) &&
                      rows16(k_cache, kv_stride_tok, kv_stride_head) &&
                      rows16(v_cache, kv_stride_block, 0),
                  LOCKS_ERR_ARG,
                  "locks_norm_rope_write: rows must be 16-byte aligned");
    LOCKS_REQUIRE(cos_sin == nullptr ||
                      (positions && n_positions >= 1 && rot_dim >= 2 &&
                       rot_dim <= head_dim && (rot_dim & 1) == 0 &&
                       cos_sin_row_stride >= rot_dim),
                  LOCKS_ERR_ARG,
                  "locks_norm_rope_write: rotation needs positions, a table and an even "
                  "rot_dim <= head_dim");
    LOCKS_REQUIRE(((reinterpret_cast<uintptr_t>(q_weight) |
                    reinterpret_cast<uintptr_t>(k_weight)) & 15) == 0,
                  LOCKS_ERR_ARG,
                  "locks_norm_rope_write: norm weights must be 16-byte aligned");
    if (n_tok == 0) return LOCKS_OK;
    NormRopeParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(key);
    p.v = static_cast<const __nv_bfloat16*>(val);
    p.q_tok = q_stride_tok; p.q_head = q_stride_head;
    p.k_tok = k_stride_tok; p.k_head = k_stride_head;
    p.v_tok = v_stride_tok; p.v_head = v_stride_head;
    p.q_out = static_cast<__nv_bfloat16*>(q_out);
    p.o_tok = o_stride_tok; p.o_head = o_stride_head;
    p.k_cache = static_cast<__nv_bfloat16*>(k_cache);
    p.v_cache = static_cast<__nv_bfloat16*>(v_cache);
    p.cb = kv_stride_block; p.ct = kv_stride_tok; p.ch = kv_stride_head;
    p.slot = slot_mapping; p.pos = positions;
    p.cos_sin = cos_sin; p.cs_row = cos_sin_row_stride;
    p.q_weight = q_weight; p.k_weight = k_weight; p.weight_f32 = weight_f32;
    p.rot = rot_dim; p.neox = neox; p.n_pos = n_positions; p.num_blocks = num_blocks;
    p.n_tok = n_tok; p.H = n_heads; p.n_kv = n_kv; p.eps = eps;
    int mode = ROPE_NONE;
    if (cos_sin) {
        // vector loads of a lane's table values: 8 (half-split) or 4 (interleaved)
        // in a row, starting at a multiple of that many and `half` behind it
        const int align = table_f32 ? 16 : 8;
        const int es = table_f32 ? 4 : 2, half = rot_dim / 2;
        const bool vec = reinterpret_cast<uintptr_t>(cos_sin) % align == 0 &&
                         (cos_sin_row_stride * es) % align == 0 &&
                         (half * es) % align == 0;
        mode = !vec ? ROPE_ANY
               : neox ? (half % 8 == 0 ? ROPE_HALVES : ROPE_ANY)
                      : (rot_dim % 8 == 0 ? ROPE_PAIRS : ROPE_ANY);
    }
    p.chunks = (n_heads + 2 * n_kv + 2 * NR_ROWS - 1) / (2 * NR_ROWS);
    constexpr int WARPS = NR_THREADS / 32;
    const dim3 grid((unsigned)(((int64_t)n_tok * p.chunks + WARPS - 1) / WARPS), 1, 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (table_f32) launch_norm_rope<float>(mode, grid, s, p);
    else launch_norm_rope<__nv_bfloat16>(mode, grid, s, p);
    return check_launch("locks_norm_rope_write");
}
