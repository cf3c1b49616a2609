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

int rope_axes(h3_gpu *g, const AxesArgs &args) {
    AxesArgs a = args;
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
