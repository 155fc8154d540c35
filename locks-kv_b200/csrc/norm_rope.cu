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
// row, 16 lanes x 8 channels, so the norm is four shuffles.  A lane's channels are eight
// in a row (one 16-byte access), or in half-split pairing four of each half (two of 8
// bytes), so that both channels of a pair are its own.  A warp takes one token
// (or, where there are few tokens, a share of its heads), whose slot, position and
// (cos | sin) row it reads once, and goes through its query, key and value heads in steps
// of NR_ROWS pairs of neighbouring rows; the next step's rows are on their way while a
// step is computed.  Pairs of channels share
// an instruction (fp32x2), which keeps the arithmetic below the memory time.
//
// Eight CTAs to an SM leave 64 registers a thread: 4 to 28 bytes spilled, 80 with ROPE_ANY.
// Where the rotated channels do not divide by eight, or the table is not aligned for
// vector loads, pairs are found one by one and meet in shared memory (ROPE_ANY): 16384
// tokens x 36 heads 81 us with 20 rotated channels and 90 with 100, against 57 with 64 or
// 128; one token x 48 heads 3.0 against 2.1.
#include <type_traits>

#include "common.cuh"

namespace locks {
namespace {

constexpr int NR_HD = 128;
constexpr int NR_THREADS = 128;
constexpr int NR_HALVES = NR_THREADS / 16;
constexpr int NR_ROWS = 2;

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
    int n_tok, H, n_kv, share, shares;             // heads of a warp, warps of a token
    float eps;
};

// two fp32 operations in one instruction
__device__ __forceinline__ float2 nr_mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float2 nr_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
          "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
// 2 N consecutive table or weight values as fp32 (N even; 8-byte aligned for bf16 and
// 16-byte for fp32)
template <int N>
__device__ __forceinline__ void load_vals(const float* p, float2 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
        f[2 * i] = make_float2(v.x, v.y);
        f[2 * i + 1] = make_float2(v.z, v.w);
    }
}
template <int N>
__device__ __forceinline__ void load_vals(const __nv_bfloat16* p, float2 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p) + i);
        f[2 * i] = unpack2(v.x);
        f[2 * i + 1] = unpack2(v.y);
    }
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <int MODE, class Tab>
__global__ void __launch_bounds__(NR_THREADS, 8) norm_rope_kernel(const NormRopeParams p) {
    __shared__ float stage[MODE == ROPE_ANY ? NR_HALVES : 1][MODE == ROPE_ANY ? NR_HD : 1];
    const int half_id = threadIdx.x >> 4, lane = threadIdx.x & 15, side = half_id & 1;
    const int heads = p.H + 2 * p.n_kv, qk = p.H + p.n_kv;
    const int job = blockIdx.x * (NR_THREADS / 32) + (threadIdx.x >> 5);
    const int t = job / p.shares;
    // launched behind the last kernel's end; the next one may line up once this one runs
    pdl_wait();
    pdl_trigger();
    if (t >= p.n_tok) return;                    // (a whole warp)
    const int h0 = (job - t * p.shares) * p.share;     // the warp's heads [h0, end)
    const int end = min(h0 + p.share, heads);
    // the lane's channels: [ca, ca + 4) and [cb, cb + 4).  Half-split: of either half
    // while there are rotated ones, the rest in order
    const int half = p.rot >> 1, quads = half >> 2;
    const bool turns = MODE == ROPE_HALVES ? lane < quads : 8 * lane < p.rot;
    const int ca = MODE != ROPE_HALVES ? 8 * lane : turns ? 4 * lane : p.rot + 8 * (lane - quads);
    const int cb = MODE == ROPE_HALVES && turns ? ca + half : ca + 4;
    auto load_row = [&](const __nv_bfloat16* row) {
        if constexpr (MODE == ROPE_HALVES) {
            const uint2 a = *reinterpret_cast<const uint2*>(row + ca);
            const uint2 b = *reinterpret_cast<const uint2*>(row + cb);
            return make_uint4(a.x, a.y, b.x, b.y);
        } else {
            return *reinterpret_cast<const uint4*>(row + ca);
        }
    };
    auto store_row = [&](__nv_bfloat16* row, const uint4 y) {
        if constexpr (MODE == ROPE_HALVES) {
            *reinterpret_cast<uint2*>(row + ca) = make_uint2(y.x, y.y);
            *reinterpret_cast<uint2*>(row + cb) = make_uint2(y.z, y.w);
        } else {
            *reinterpret_cast<uint4*>(row + ca) = y;
        }
    };
    const int64_t slot = p.slot[t];
    // the token's table row, as far as this lane's channels need it
    const Tab* cs = static_cast<const Tab*>(p.cos_sin);
    float2 c[4], s[4];
    if constexpr (MODE != ROPE_NONE) {
        cs += min(max(p.pos[t], (int64_t)0), (int64_t)p.n_pos - 1) * p.cs_row;
        if ((MODE == ROPE_PAIRS || MODE == ROPE_HALVES) && turns) {
            float2 (&c2)[2] = reinterpret_cast<float2 (&)[2]>(c);
            float2 (&s2)[2] = reinterpret_cast<float2 (&)[2]>(s);
            load_vals(cs + 4 * lane, c2);
            load_vals(cs + half + 4 * lane, s2);
        }
        if (MODE == ROPE_ANY) {                  // any even rot, any alignment
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                auto pair = [&](int d, float& ce, float& se) {
                    const bool first = p.neox ? d < half : (d & 1) == 0;
                    const int j = p.neox ? (first ? d : d - half) : d >> 1;
                    ce = d < p.rot ? to_f32(cs[j]) : 1.f;
                    se = d < p.rot ? to_f32(cs[half + j]) : 0.f;
                    if (first) se = -se;
                };
                pair(8 * lane + 2 * e, c[e].x, s[e].x);
                pair(8 * lane + 2 * e + 1, c[e].y, s[e].y);
            }
        }
    }
    const bool stored = slot >= 0 && (slot >> 4) < p.num_blocks;
    const int64_t at = stored ? (slot >> 4) * p.cb + (slot & 15) * p.ct : 0;
    // Heads [from, to) of one kind: rows `src_step` / `dst_step` apart, the half-warp's own
    // every second one.  turn: norm (with a weight) and rotation, else a copy.
    auto heads_of = [&](auto turn, int from, int to, const __nv_bfloat16* src, int64_t src_step,
                        __nv_bfloat16* dst, int64_t dst_step, const void* weight, bool store) {
        if (from >= to) return;
        const int mine = (to - from - side + 1) >> 1, pairs = (to - from + 1) >> 1;
        src += side * src_step;
        dst += side * dst_step;
        src_step *= 2;
        dst_step *= 2;
        float2 w[4];
        if (decltype(turn)::value && weight) {
            float2 (&wa)[2] = reinterpret_cast<float2 (&)[2]>(w[0]);
            float2 (&wb)[2] = reinterpret_cast<float2 (&)[2]>(w[2]);
            if (p.weight_f32) {
                load_vals(static_cast<const float*>(weight) + ca, wa);
                load_vals(static_cast<const float*>(weight) + cb, wb);
            } else {
                load_vals(static_cast<const __nv_bfloat16*>(weight) + ca, wa);
                load_vals(static_cast<const __nv_bfloat16*>(weight) + cb, wb);
            }
        }
        uint4 next[NR_ROWS];
#pragma unroll
        for (int i = 0; i < NR_ROWS; ++i) {
            next[i] = make_uint4(0, 0, 0, 0);
            if (i < mine) next[i] = load_row(src + i * src_step);
        }
        for (int j = 0; j < pairs; j += NR_ROWS) {
            uint4 x[NR_ROWS];
#pragma unroll
            for (int i = 0; i < NR_ROWS; ++i) x[i] = next[i];
            src += NR_ROWS * src_step;
#pragma unroll
            for (int i = 0; i < NR_ROWS; ++i)
                if (j + NR_ROWS + i < mine) next[i] = load_row(src + i * src_step);
#pragma unroll
            for (int i = 0; i < NR_ROWS; ++i) {
                // (both half-warps come along: the shuffles need all lanes)
                uint4 y = x[i];
                if constexpr (decltype(turn)::value) {
                    const uint32_t raw[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    float2 f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = unpack2(raw[e]);
                    if (weight) {
                        float2 sq = nr_mul2(f[0], f[0]);
#pragma unroll
                        for (int e = 1; e < 4; ++e) sq = nr_fma2(f[e], f[e], sq);
                        float ss = sq.x + sq.y;
#pragma unroll
                        for (int d = 1; d < 16; d <<= 1)
                            ss += __shfl_xor_sync(0xffffffffu, ss, d);
                        const float rs = rsqrtf(ss * (1.f / NR_HD) + p.eps);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            f[e] = nr_mul2(nr_mul2(f[e], make_float2(rs, rs)), w[e]);
                    }
                    if constexpr (MODE == ROPE_PAIRS) {
                        if (turns) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float ce = e & 1 ? c[e >> 1].y : c[e >> 1].x;
                                const float se = e & 1 ? s[e >> 1].y : s[e >> 1].x;
                                f[e] = nr_fma2(make_float2(f[e].y, f[e].x), make_float2(-se, se),
                                               nr_mul2(f[e], make_float2(ce, ce)));
                            }
                        }
                    } else if constexpr (MODE == ROPE_HALVES) {
                        if (turns) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float2 a = f[e], b = f[2 + e];
                                f[e] = nr_fma2(b, make_float2(-s[e].x, -s[e].y), nr_mul2(a, c[e]));
                                f[2 + e] = nr_fma2(a, s[e], nr_mul2(b, c[e]));
                            }
                        }
                    } else if constexpr (MODE == ROPE_ANY) {
                        // the partner of a channel may sit in any lane: through shared memory
                        float* row = stage[half_id];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<float2*>(&row[8 * lane + 2 * e]) = f[e];
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            auto partner = [&](int d) {
                                return !p.neox ? d ^ 1 : d < half ? d + half : d - half;
                            };
                            const int d = 8 * lane + 2 * e;
                            if (d >= p.rot) break;          // (rot is even)
                            f[e] = nr_fma2(make_float2(row[partner(d)], row[partner(d + 1)]),
                                           s[e], nr_mul2(f[e], c[e]));
                        }
                        __syncwarp();
                    }
                    y = make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y),
                                   pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y));
                }
                if (store && j + i < mine) store_row(dst + i * dst_step, y);
            }
            dst += NR_ROWS * dst_step;
        }
    };
    const int64_t tq = t * p.q_tok, to = t * p.o_tok, tk = t * p.k_tok, tv = t * p.v_tok;
    const int k0 = max(h0, p.H), v0 = max(h0, qk);
    heads_of(std::true_type{}, h0, min(end, p.H), p.q + tq + h0 * p.q_head, p.q_head,
             p.q_out + to + h0 * p.o_head, p.o_head, p.q_weight, true);
    heads_of(std::true_type{}, k0, min(end, qk), p.k + tk + (k0 - p.H) * p.k_head, p.k_head,
             p.k_cache + at + (k0 - p.H) * p.ch, p.ch, p.k_weight, stored);
    heads_of(std::false_type{}, v0, end, p.v + tv + (v0 - qk) * p.v_head, p.v_head,
             p.v_cache + at + (v0 - qk) * p.ch, p.ch, nullptr, stored);
}

template <class Tab>
cudaError_t launch_norm_rope(int mode, dim3 grid, cudaStream_t s, const NormRopeParams& p) {
    void (*kernel)(const NormRopeParams) =
        mode == ROPE_NONE ? norm_rope_kernel<ROPE_NONE, Tab>
        : mode == ROPE_PAIRS ? norm_rope_kernel<ROPE_PAIRS, Tab>
        : mode == ROPE_HALVES ? norm_rope_kernel<ROPE_HALVES, Tab>
                              : norm_rope_kernel<ROPE_ANY, Tab>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(NR_THREADS, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, p);
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
        // vector loads of a lane's table values: four in a row, starting at a multiple
        // of four and `half` behind it
        const int align = table_f32 ? 16 : 8;
        const int es = table_f32 ? 4 : 2, half = rot_dim / 2;
        const bool vec = reinterpret_cast<uintptr_t>(cos_sin) % align == 0 &&
                         (cos_sin_row_stride * es) % align == 0 &&
                         (half * es) % align == 0;
        mode = !vec || rot_dim % 8 != 0 ? ROPE_ANY : neox ? ROPE_HALVES : ROPE_PAIRS;
    }
    // A token to a warp when that fills the device about once (32 warps to an SM); else
    // its heads are shared by more warps, down to one step each.  16384 tokens x 36 heads:
    // 58 us (5.3 TB/s) with a token to a warp, 75 with a step to a warp; 2053 tokens x 48
    // heads: 15.9 us with two steps to a warp, 18.3 with a token.
    constexpr int WARPS = NR_THREADS / 32, STEP = 2 * NR_ROWS;
    const int heads = n_heads + 2 * n_kv, steps = (heads + STEP - 1) / STEP;
    int per = steps;
    while (per > 1 && (int64_t)n_tok * ((steps + per - 1) / per) < (int64_t)sm_count() * 32)
        per = (per + 1) / 2;
    p.share = per * STEP;
    p.shares = (steps + per - 1) / per;
    const dim3 grid((unsigned)(((int64_t)n_tok * p.shares + WARPS - 1) / WARPS), 1, 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = table_f32 ? launch_norm_rope<float>(mode, grid, s, p)
                                    : launch_norm_rope<__nv_bfloat16>(mode, grid, s, p);
    if (e != cudaSuccess)
        return fail(LOCKS_ERR_LAUNCH, "locks_norm_rope_write: %s", cudaGetErrorString(e));
    return check_launch("locks_norm_rope_write");
}
