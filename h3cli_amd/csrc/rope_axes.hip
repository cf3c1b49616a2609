// Per-head RMSNorm of Q and K and their rotation by positions of several axes, from fused
// QKV rows, in one pass (h3_hip_qkv_rope_axes_bf16). The rows may belong to any requests:
// each brings its own position on every axis.
//
//   x' = x * rsqrt(mean(x^2) + eps) * w            (over the head's channels; optional)
//   angle_j = position[row, axis_j] * f_j
//   (a, b) -> (a cos - b sin, b cos + a sin)        a, b: channels j and j + pairs, or 2 j and 2 j + 1
//
// All in FP32, one rounding to BF16. The pass is bound by HBM (4 bytes a value), so the
// rotation must stay below the loads: cosines and sines are made once per row and channel
// and kept in registers for all heads, with the norm's weights folded into them:
//   x'_d cos +- x'_p sin = r (x_d (w_d cos) + x_p (+-w_p sin)),   r the head's norm factor.
//
// Angles. A position may be far (2^24 and beyond), where an FP32 angle has lost its phase. With
// f / 2 pi = hi + lo in two floats, n = rint(p hi), the phase in turns is
//   fma(p, lo, fma(p, hi, -n)),
// whose inner fma is exact but for one rounding of a value of at most a half (2^-25 turns); the
// hardware's sine and cosine take turns.
#include "common.h"
#include "internal.h"
#include <algorithm>
#include <new>
#include <vector>

struct h3_hip_rope_axes {
    h3_gpu *owner;
    h3_gpu_tensor *table;    // F32 [pairs][2]: f / 2 pi in two floats; then the axis of each pair (u32 bits)
    uint32_t pairs, axes;
    int interleaved;
};

namespace {

struct AxesArgs {
    uint16_t *q, *k, *v;
    const uint16_t *qkv, *qw, *kw;
    const float *turns;          // [pairs][2]
    const uint32_t *axis;        // [pairs]
    const float *positions;      // [rows][axes]
    unsigned rows, heads, kv_heads, dim, pairs, axes, splits;
    float eps;
    int grouped, interleaved;
};

enum Kind { QUERY, KEY, VALUE };

// Item i of a row's heads, queries first, then keys, then values: its source head within the
// row, its head within its own output.
__device__ inline unsigned source_head(const AxesArgs &a, unsigned i, unsigned &head, int &kind) {
    kind = i < a.heads ? QUERY : i < a.heads + a.kv_heads ? KEY : VALUE;
    head = kind == QUERY ? i : kind == KEY ? i - a.heads : i - a.heads - a.kv_heads;
    if (!a.grouped) return i;
    const unsigned share = a.heads / a.kv_heads;
    return kind == QUERY ? head / share * (share + 2) + head % share : head * (share + 2) + share + (kind == VALUE);
}

__device__ inline void phase(const AxesArgs &a, size_t row, unsigned pair, float &c, float &s) {
    const float p = a.positions[row * a.axes + a.axis[pair]];
    const float hi = a.turns[2 * pair], lo = a.turns[2 * pair + 1];
    const float t = fmaf(p, lo, fmaf(p, hi, -rintf(p * hi)));
    c = __builtin_amdgcn_cosf(t);
    s = __builtin_amdgcn_sinf(t);
}

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Any head width up to 256 and any number of pairs: a wave per head, two channels a lane and
// 128 channels a step; partners go through LDS.
__global__ __launch_bounds__(256) void rope_axes_any(AxesArgs a) {
    __shared__ float stage[4][256];
    const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const unsigned items = a.heads + 2 * a.kv_heads;
    const bool wide = a.dim % 2 == 0;                      // every head then starts on four bytes
    for (size_t block = blockIdx.x; block < (size_t)a.rows * a.splits; block += gridDim.x) {
        const size_t row = block / a.splits;
        const unsigned part = block % a.splits;
        // Channel d = 128 i + 2 lane + e: its partner and the factors of both.
        unsigned partner[2][2];
        float own[2][2], other[2][2];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const unsigned d = 128 * i + 2 * lane + e;
                partner[i][e] = min(d, a.dim - 1);
                own[i][e] = 1.f;
                other[i][e] = 0.f;
                if (d < 2 * a.pairs) {
                    const bool second = a.interleaved ? d % 2 : d >= a.pairs;
                    const unsigned pair = a.interleaved ? d / 2 : second ? d - a.pairs : d;
                    phase(a, row, pair, own[i][e], other[i][e]);
                    if (!second) other[i][e] = -other[i][e];
                    partner[i][e] = a.interleaved ? d ^ 1 : second ? d - a.pairs : d + a.pairs;
                }
            }
        for (unsigned item = part * 4 + wave; item < items; item += a.splits * 4) {
            unsigned head;
            int kind;
            const unsigned from = source_head(a, item, head, kind);
            const uint16_t *src = a.qkv + (row * items + from) * a.dim;
            uint16_t *dst = kind == QUERY ? a.q + (row * a.heads + head) * a.dim
                                          : (kind == KEY ? a.k : a.v) + (row * a.kv_heads + head) * a.dim;
            const uint16_t *w = kind == QUERY ? a.qw : kind == KEY ? a.kw : nullptr;
            uint16_t raw[2][2] = {};
            float x[2][2], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const unsigned d = 128 * i + 2 * lane;
                if (d >= a.dim) continue;
                if (wide) {
                    const uint32_t both = *reinterpret_cast<const uint32_t *>(src + d);
                    raw[i][0] = both & 0xffff;
                    raw[i][1] = both >> 16;
                } else {
                    raw[i][0] = src[d];
                    if (d + 1 < a.dim) raw[i][1] = src[d + 1];
                }
            }
            if (kind != VALUE) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const unsigned d = 128 * i + 2 * lane + e;
                        x[i][e] = bf16_to_f32(raw[i][e]);
                        sum = fmaf(x[i][e], x[i][e], sum);
                        if (w && d < a.dim) x[i][e] *= bf16_to_f32(w[d]);
                        stage[wave][d] = x[i][e];
                    }
                const float r = w ? rsqrtf(wave_sum(sum) / (float)a.dim + a.eps) : 1.f;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own stores
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                    {
                        // Channels behind the pairs pass as they are, infinities too.
                        const bool turned = 128 * i + 2 * lane + e < 2 * a.pairs;
                        raw[i][e] = f32_to_bf16(r * (turned ? fmaf(x[i][e], own[i][e], stage[wave][partner[i][e]] * other[i][e])
                                                            : x[i][e]));
                    }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next head's
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const unsigned d = 128 * i + 2 * lane;
                if (d >= a.dim) continue;
                if (wide) *reinterpret_cast<uint32_t *>(dst + d) = raw[i][0] | (uint32_t)raw[i][1] << 16;
                else {
                    dst[d] = raw[i][0];
                    if (d + 1 < a.dim) dst[d + 1] = raw[i][1];
                }
            }
        }
    }
}

// Sums over the 16 / 8 / 32 lanes of a head by row rotations of the VALU; every lane gets the
// same bits, since both sides of each addition are the same two values.
template <int CTRL> __device__ inline float rotated(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LANES> __device__ inline float head_sum(float v) {
    static_assert(LANES >= 1 && LANES <= 32, "lanes of a head");
    if constexpr (LANES >= 2) v += rotated<0xb1>(v);                    // quad_perm [1, 0, 3, 2]
    if constexpr (LANES >= 4) v += rotated<0x4e>(v);                    // quad_perm [2, 3, 0, 1]
    if constexpr (LANES >= 8) v += rotated<0x141>(v);                   // row_half_mirror
    if constexpr (LANES >= 16) v += rotated<0x140>(v);                  // row_mirror
    if constexpr (LANES >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

// Heads of 8 * CHUNKS channels, CHUNKS <= LANES a power of two: LANES lanes a head, a 16-byte chunk each.
// A workgroup takes a row (or a share of its heads) and goes through the heads 256 / LANES at
// a time, UNROLL of them in flight a lane. Pairs of halves need pairs % 8 == 0 (a chunk's partner
// is a chunk, fetched from its lane), interleaved ones pairs % 4 == 0 (partners are in the chunk).
template <int LANES, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_axes_chunks(AxesArgs a) {
    constexpr int GROUPS = 256 / LANES, UNROLL = 4;
    const unsigned lane = threadIdx.x % 64, c = lane % LANES, group = threadIdx.x / LANES;
    const unsigned items = a.heads + 2 * a.kv_heads, chunks = a.dim / 8;
    const bool held = c < chunks;
    const unsigned half = INTERLEAVED ? 0 : a.pairs / 8;
    const bool turned = INTERLEAVED ? c < a.pairs / 4 : c < 2 * half;
    const bool second = !INTERLEAVED && c >= half;
    const int partner = (int)(turned && !INTERLEAVED ? lane + (second ? 0u - half : half) : lane) * 4;
    const float inv_dim = 1.f / (float)a.dim;
    u16x8 wq{}, wk{}, pq{}, pk{};
    if (a.qw && held) {
        const unsigned pc = turned && !INTERLEAVED ? (second ? c - half : c + half) : c;
        wq = *reinterpret_cast<const u16x8 *>(a.qw + c * 8);
        wk = *reinterpret_cast<const u16x8 *>(a.kw + c * 8);
        pq = *reinterpret_cast<const u16x8 *>(a.qw + pc * 8);
        pk = *reinterpret_cast<const u16x8 *>(a.kw + pc * 8);
    }
    for (size_t block = blockIdx.x; block < (size_t)a.rows * a.splits; block += gridDim.x) {
        const size_t row = block / a.splits;
        const unsigned part = block % a.splits;
        // Channel e of the chunk: what it and its partner are multiplied with.
        float oq[8], tq[8], ok[8], tk[8];
        {
            float cs[8], sn[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                cs[e] = 1.f;
                sn[e] = 0.f;
            }
            if (turned) {
#pragma unroll
                for (int e = 0; e < 8; e += INTERLEAVED ? 2 : 1) {
                    const unsigned pair = INTERLEAVED ? c * 4 + e / 2 : (second ? c - half : c) * 8 + e;
                    phase(a, row, pair, cs[e], sn[e]);
                    if constexpr (INTERLEAVED) {
                        cs[e + 1] = cs[e];
                        sn[e + 1] = sn[e];
                        sn[e] = -sn[e];
                    } else if (!second) {
                        sn[e] = -sn[e];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int pe = INTERLEAVED ? e ^ 1 : e;
                oq[e] = a.qw ? cs[e] * bf16_to_f32(wq[e]) : cs[e];
                ok[e] = a.qw ? cs[e] * bf16_to_f32(wk[e]) : cs[e];
                tq[e] = a.qw ? sn[e] * bf16_to_f32(pq[pe]) : sn[e];
                tk[e] = a.qw ? sn[e] * bf16_to_f32(pk[pe]) : sn[e];
            }
        }
        const uint16_t *const src = a.qkv + row * items * a.dim + c * 8;
        for (unsigned first = part * GROUPS + group; first < items; first += a.splits * GROUPS * UNROLL) {
            u16x8 raw[UNROLL] = {};
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const unsigned item = first + u * a.splits * GROUPS;
                unsigned head;
                int kind;
                if (item < items && held)
                    raw[u] = *reinterpret_cast<const u16x8 *>(src + (size_t)source_head(a, item, head, kind) * a.dim);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const unsigned item = first + u * a.splits * GROUPS;
                if (item >= items) break;
                unsigned head;
                int kind;
                source_head(a, item, head, kind);
                uint16_t *const dst = (kind == QUERY ? a.q + (row * a.heads + head) * a.dim
                                                     : (kind == KEY ? a.k : a.v) + (row * a.kv_heads + head) * a.dim) + c * 8;
                if (kind != VALUE) {
                    float x[8], sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = bf16_to_f32(raw[u][e]);
                        sum = fmaf(x[e], x[e], sum);
                    }
                    const float r = a.qw ? rsqrtf(head_sum<LANES>(sum) * inv_dim + a.eps) : 1.f;
                    float y[8];
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int e = 0; e < 8; e++) y[e] = turned ? x[e ^ 1] : 0.f;
                    } else {
                        const i32x4 own = __builtin_bit_cast(i32x4, raw[u]);
                        i32x4 other;
#pragma unroll
                        for (int e = 0; e < 4; e++) other[e] = __builtin_amdgcn_ds_bpermute(partner, own[e]);
                        // Channels behind the pairs pass as they are, infinities too.
#pragma unroll
                        for (int e = 0; e < 4; e++) other[e] = turned ? other[e] : 0;
                        const u16x8 o = __builtin_bit_cast(u16x8, other);
#pragma unroll
                        for (int e = 0; e < 8; e++) y[e] = bf16_to_f32(o[e]);
                    }
                    if (kind == QUERY)
#pragma unroll
                        for (int e = 0; e < 8; e++) raw[u][e] = f32_to_bf16(r * fmaf(x[e], oq[e], y[e] * tq[e]));
                    else
#pragma unroll
                        for (int e = 0; e < 8; e++) raw[u][e] = f32_to_bf16(r * fmaf(x[e], ok[e], y[e] * tk[e]));
                }
                if (held) *reinterpret_cast<u16x8 *>(dst) = raw[u];
            }
        }
    }
}

template <int LANES> void launch_chunks(h3_gpu *g, AxesArgs a) {
    const unsigned items = a.heads + 2 * a.kv_heads;
    constexpr unsigned GROUPS = 256 / LANES;
    // A row's heads go to more workgroups where the rows alone would not fill the chip.
    a.splits = (unsigned)std::min<size_t>((items + GROUPS - 1) / GROUPS, (2048 + (size_t)a.rows - 1) / a.rows);
    const unsigned blocks = (unsigned)std::min<size_t>((size_t)a.rows * a.splits, 1 << 20);
    if (a.interleaved) hipLaunchKernelGGL((rope_axes_chunks<LANES, true>), dim3(blocks), dim3(256), 0, g->compute, a);
    else hipLaunchKernelGGL((rope_axes_chunks<LANES, false>), dim3(blocks), dim3(256), 0, g->compute, a);
}

int rope_axes(h3_gpu *g, const AxesArgs &args) {
    AxesArgs a = args;
    if (a.dim % 8 == 0 && a.pairs % (a.interleaved ? 4 : 8) == 0) {
        const unsigned chunks = a.dim / 8;
        if (chunks <= 2) launch_chunks<2>(g, a);
        else if (chunks <= 4) launch_chunks<4>(g, a);
        else if (chunks <= 8) launch_chunks<8>(g, a);
        else if (chunks <= 16) launch_chunks<16>(g, a);
        else launch_chunks<32>(g, a);
        return h3_launch_status(g, "QKV norm/RoPE by axes");
    }
    const unsigned items = a.heads + 2 * a.kv_heads;
    // A row's heads go to more workgroups where the rows alone would not fill the chip.
    a.splits = (unsigned)std::min<size_t>((items + 3) / 4, (4096 + (size_t)a.rows - 1) / a.rows);
    const size_t blocks = std::min<size_t>((size_t)a.rows * a.splits, 1 << 20);
    hipLaunchKernelGGL(rope_axes_any, dim3((unsigned)blocks), dim3(256), 0, g->compute, a);
    return h3_launch_status(g, "QKV norm/RoPE by axes");
}

}  // namespace

extern "C" void h3_hip_rope_axes_free(h3_hip_rope_axes *r) {
    if (!r) return;
    h3_gpu_tensor_free(r->table);
    delete r;
}

extern "C" h3_hip_rope_axes *h3_hip_rope_axes_new(h3_gpu *g, const double *frequencies, const uint32_t *axis, uint32_t pairs,
                                                  uint32_t axes, int interleaved) {
    if (!g) return nullptr;
    if (!frequencies || !axis || !pairs || pairs > 128 || !axes || axes > 16 || (interleaved != 0 && interleaved != 1)) {
        h3_set_error(g, "RoPE axes: need 1 to 128 pairs of 1 to 16 axes, their frequencies, and interleaved 0 or 1");
        return nullptr;
    }
    float words[128 * 3] = {};
    for (uint32_t j = 0; j < pairs; j++) {
        const double turns = frequencies[j] / 6.283185307179586476925;
        if (axis[j] >= axes || !finite_f32((float)frequencies[j])) {
            h3_set_error(g, "RoPE axes: pair %u has axis %u of %u or a frequency that is not finite", j, axis[j], axes);
            return nullptr;
        }
        words[2 * j] = (float)turns;
        words[2 * j + 1] = (float)(turns - (double)words[2 * j]);
        memcpy(&words[2 * pairs + j], &axis[j], 4);
    }
    auto *r = new (std::nothrow) h3_hip_rope_axes{g, nullptr, pairs, axes, interleaved};
    if (!r) { h3_set_error(g, "RoPE axes: out of host memory"); return nullptr; }
    r->table = h3_gpu_tensor_from_f32(g, words, (size_t)pairs * 3);
    if (!r->table) { delete r; return nullptr; }
    return r;
}

extern "C" int h3_hip_qkv_rope_axes_bf16(h3_gpu *g, h3_gpu_tensor *q, h3_gpu_tensor *k, h3_gpu_tensor *v,
                                         const h3_gpu_tensor *qkv, const h3_gpu_tensor *qw, const h3_gpu_tensor *kw,
                                         const h3_hip_rope_axes *rope, const h3_gpu_tensor *positions, uint32_t rows,
                                         uint32_t heads, uint32_t kv_heads, uint32_t dim, int grouped, float eps) {
    if (!h3_launch_ready(g)) return 0;
    if (!rope || rope->owner != g) return h3_set_error(g, "QKV RoPE by axes: missing axes, or of another context");
    if (!rows || !heads || !kv_heads || heads > 65535 || heads % kv_heads || !dim || dim > 256 || rope->pairs * 2 > dim ||
        !qw != !kw || (grouped != 0 && grouped != 1) || !finite_f32(eps) || eps < 0)
        return h3_set_error(g, "QKV RoPE by axes: need rows, heads a multiple of the key heads, dim <= 256, 2 * pairs <= dim, "
                               "both or neither norm weights, grouped 0 or 1 and eps >= 0");
    const size_t nq = (size_t)rows * heads * dim, nk = (size_t)rows * kv_heads * dim;
    if (!h3_require(g, qkv, H3_GPU_BF16, nq + 2 * nk, "QKV") || !h3_require(g, q, H3_GPU_BF16, nq, "Q") ||
        !h3_require(g, k, H3_GPU_BF16, nk, "K") || !h3_require(g, v, H3_GPU_BF16, nk, "V") ||
        (qw && (!h3_require(g, qw, H3_GPU_BF16, dim, "Q norm") || !h3_require(g, kw, H3_GPU_BF16, dim, "K norm"))) ||
        !h3_require(g, positions, H3_GPU_F32, (size_t)rows * rope->axes, "RoPE positions"))
        return 0;
    if (q == qkv || k == qkv || v == qkv || q == k || q == v || k == v)
        return h3_set_error(g, "QKV RoPE by axes: outputs and input must be disjoint");
    const AxesArgs a{(uint16_t *)q->data, (uint16_t *)k->data, (uint16_t *)v->data, (const uint16_t *)qkv->data,
                     qw ? (const uint16_t *)qw->data : nullptr, kw ? (const uint16_t *)kw->data : nullptr,
                     (const float *)rope->table->data, (const uint32_t *)rope->table->data + 2 * rope->pairs,
                     (const float *)positions->data, rows, heads, kv_heads, dim, rope->pairs, rope->axes, 1, eps, grouped,
                     rope->interleaved};
    return rope_axes(g, a);
}
