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
// and kept in LDS for all its heads, with the norms' weights folded into them:
//   x'_d cos +- x'_p sin = r (x_d (w_d cos) + x_p (+-w_p sin)),   r the head's norm factor.
//
// Angles. A position may be far (2^24 and beyond), where an FP32 angle has lost its phase. With
// f / 2 pi = hi + lo in two floats, the phase in turns is
//   near = fma(p, hi, -rint(p hi)),   t = fma(p, lo, near - rint(near)),   t - rint(t).
// Up to 2^24 turns near is below one turn and off by half a bit of that, 2^-25; beyond, it is what p hi
// was rounded by, exactly, and may be many turns. p lo is off by lo's rounding, 2^-48 of the angle, and t by its
// own. In all up to 2^24 turns 2^-23 turns, beyond them 2^-47 of the angle. The hardware's sine and cosine
// take turns, up to 256 of them: t alone passes that at 2^33 turns, and is brought below half a turn.
#include "common.h"
#include "internal.h"
#include <algorithm>
#include <new>
#include <type_traits>
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
    unsigned rows, heads, kv_heads, share, dim, pairs, axes, splits, together;
    float eps;
    int grouped, interleaved;
};

enum Kind { QUERY, KEY, VALUE };

// Head i of rows from row0 on, each row's queries first, then its keys and values.
struct Item {
    int kind;
    unsigned row, from, to;   // its row, and its first channel in qkv and in its own output, behind row0's
};
__device__ inline Item item_of(const AxesArgs &a, unsigned i, unsigned items) {
    const unsigned row = a.together == 1 ? 0 : i / items, h = i - row * items;
    const int kind = h < a.heads ? QUERY : h < a.heads + a.kv_heads ? KEY : VALUE;
    const unsigned head = kind == QUERY ? h : kind == KEY ? h - a.heads : h - a.heads - a.kv_heads;
    const unsigned source = !a.grouped        ? h
                            : kind == QUERY ? head / a.share * (a.share + 2) + head % a.share
                                            : head * (a.share + 2) + a.share + (kind == VALUE);
    return {kind, row, (row * items + source) * a.dim, (row * (kind == QUERY ? a.heads : a.kv_heads) + head) * a.dim};
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

// Eight values from any element on. Global memory takes 16-byte accesses at any two bytes; what
// lies behind a tensor's end is within its allocation.
// Values stay packed, two a register, until they are used.
struct __attribute__((packed, aligned(2))) Loose { i32x4 v; };
__device__ inline i32x4 load_loose(const uint16_t *p) { return reinterpret_cast<const Loose *>(p)->v; }
__device__ inline float value(const i32x4 &v, int e) {
    return __builtin_bit_cast(float, e % 2 ? (uint32_t)v[e / 2] & 0xffff0000u : (uint32_t)v[e / 2] << 16);
}
__device__ inline void put(i32x4 &v, int e, uint16_t bits) { v[e / 2] |= (uint32_t)bits << (e % 2 * 16); }

// How a channel finds its partner.
enum Pairing {
    HALVES,          // j and j + pairs, pairs % 8 == 0: a chunk's partner is another lane's chunk
    HALVES_LOOSE,    // any number of pairs: loaded again, from the caches
    NEIGHBOURS,      // 2 j and 2 j + 1: in the chunk
};

// LANES lanes a head, a chunk of eight channels each (the last one cut off where the head ends).
// A workgroup takes `together` rows at a time (more than one where a row's heads would leave lanes
// idle), or a share of a row's heads, and goes through their queries, keys and values 256 / LANES at a
// time, UNROLL of them in flight a lane. Thread d makes what channel d and its partner are multiplied
// with in the next rows, the norms' weights included, while these rows' heads are on their way;
// lanes take their chunk's from LDS.
constexpr unsigned TOGETHER = 4;
template <int LANES, Pairing PAIRING>
__global__ __launch_bounds__(256, 5) void rope_axes_chunks(AxesArgs a) {
    constexpr int GROUPS = 256 / LANES, UNROLL = PAIRING == HALVES_LOOSE ? 2 : 4;   // in five waves' registers
    extern __shared__ __attribute__((aligned(16))) float factors[];   // [buffer][row][query, key][channel, partner][256]
    const unsigned tid = threadIdx.x, lane = tid % 64, c = lane % LANES, d0 = c * 8, group = tid / LANES;
    const unsigned items = a.heads + 2 * a.kv_heads;
    const bool held = d0 < a.dim, whole = d0 + 8 <= a.dim;
    const float inv_dim = 1.f / (float)a.dim;
    // Channel tid: its pair, whether it is the pair's first, its partner.
    const bool turns = tid < 2 * a.pairs, first_channel = PAIRING == NEIGHBOURS ? tid % 2 == 0 : tid < a.pairs;
    const unsigned pair = PAIRING == NEIGHBOURS ? tid / 2 : first_channel ? tid : tid - a.pairs;
    const unsigned partner_channel = !turns ? tid : PAIRING == NEIGHBOURS ? tid ^ 1 : first_channel ? tid + a.pairs : tid - a.pairs;
    float hi = 0.f, lo = 0.f, weight[2] = {1.f, 1.f}, partner_weight[2] = {1.f, 1.f};
    unsigned axis = 0;
    if (turns) {
        hi = a.turns[2 * pair];
        lo = a.turns[2 * pair + 1];
        axis = a.axis[pair];
    }
    if (a.qw && tid < a.dim) {
        weight[QUERY] = bf16_to_f32(a.qw[tid]);
        weight[KEY] = bf16_to_f32(a.kw[tid]);
        partner_weight[QUERY] = bf16_to_f32(a.qw[partner_channel]);
        partner_weight[KEY] = bf16_to_f32(a.kw[partner_channel]);
    }
    // Task: `together` rows, or a share of one row.
    const size_t tasks = ((size_t)a.rows + a.together - 1) / a.together * a.splits;
    float next[TOGETHER] = {};
    auto positions = [&](size_t task) {
#pragma unroll
        for (unsigned r = 0; r < TOGETHER; r++) {
            const size_t row = task / a.splits * a.together + r;
            if (r < a.together && turns && row < a.rows) next[r] = a.positions[row * a.axes + axis];
        }
    };
    auto turn = [&](unsigned buffer) {
#pragma unroll
        for (unsigned r = 0; r < TOGETHER; r++) {
            if (r >= a.together) break;
            const float near = fmaf(next[r], hi, -rintf(next[r] * hi)), far = fmaf(next[r], lo, near - rintf(near)), t = far - rintf(far);
            const float cs = turns ? __builtin_amdgcn_cosf(t) : 1.f, sn = turns ? __builtin_amdgcn_sinf(t) : 0.f;
#pragma unroll
            for (int kind = QUERY; kind <= KEY; kind++) {
                float *const f = factors + ((buffer * a.together + r) * 2 + kind) * 512 + tid;
                f[0] = cs * weight[kind];
                f[256] = (first_channel ? -sn : sn) * partner_weight[kind];
            }
        }
    };
    positions(blockIdx.x);
    turn(0);
    __syncthreads();
    unsigned buffer = 0;
    for (size_t task = blockIdx.x; task < tasks; task += gridDim.x, buffer ^= 1) {
        const size_t row0 = task / a.splits * a.together;
        const unsigned part = task % a.splits, count = (unsigned)min((size_t)a.together, a.rows - row0) * items;
        positions(task + gridDim.x);
        const uint16_t *const qkv = a.qkv + row0 * items * a.dim;
        uint16_t *const q = a.q + row0 * a.heads * a.dim, *const k = a.k + row0 * a.kv_heads * a.dim, *const v = a.v + row0 * a.kv_heads * a.dim;
        for (unsigned first = part * GROUPS + group; first < count; first += a.splits * GROUPS * UNROLL) {
            i32x4 raw[UNROLL] = {}, up[UNROLL] = {}, low[UNROLL] = {};
            Item at[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                at[u] = item_of(a, first + u * a.splits * GROUPS, items);
                if (first + u * a.splits * GROUPS >= count || !held) continue;
                const unsigned from = at[u].from + d0;
                raw[u] = load_loose(qkv + from);
                if (PAIRING == HALVES_LOOSE && at[u].kind != VALUE) {
                    if (d0 < a.pairs) up[u] = load_loose(qkv + from + a.pairs);
                    if (d0 + 7 >= a.pairs && d0 < 2 * a.pairs) {
                        if (row0 || from >= a.pairs) low[u] = load_loose(qkv + from - a.pairs);
                        else   // the very first head's chunk across the middle: its partners start behind the tensor's first value
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (from + e >= a.pairs) put(low[u], e, qkv[from + e - a.pairs]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                if (first + u * a.splits * GROUPS >= count) break;
                if (at[u].kind != VALUE) {
                    const f32x4 *const f = reinterpret_cast<const f32x4 *>(factors + ((buffer * a.together + at[u].row) * 2 + at[u].kind) * 512 + d0);
                    const f32x4 own[2] = {f[0], f[1]}, other[2] = {f[64], f[65]};
                    float x[8], y[8], sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = PAIRING == HALVES || d0 + e < a.dim ? value(raw[u], e) : 0.f;
                        sum = fmaf(x[e], x[e], sum);
                    }
                    const float r = a.qw ? rsqrtf(head_sum<LANES>(sum) * inv_dim + a.eps) : 1.f;
                    if constexpr (PAIRING == HALVES) {
                        const bool turned = d0 < 2 * a.pairs;
                        const int partner = (int)(turned ? d0 < a.pairs ? lane + a.pairs / 8 : lane - a.pairs / 8 : lane) * 4;
                        i32x4 theirs;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            theirs[e] = __builtin_amdgcn_ds_bpermute(partner, raw[u][e]);
                            theirs[e] = turned ? theirs[e] : 0;
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) y[e] = value(theirs, e);
                    } else {
                        // Channels behind the pairs pass as they are, infinities too.
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const unsigned d = d0 + e;
                            const float theirs = PAIRING == NEIGHBOURS ? x[e ^ 1] : d < a.pairs ? value(up[u], e) : value(low[u], e);
                            y[e] = d < 2 * a.pairs ? theirs : 0.f;
                        }
                    }
                    bf16x8 result;
#pragma unroll
                    for (int e = 0; e < 8; e++) result[e] = (__bf16)(r * fmaf(x[e], own[e / 4][e % 4], y[e] * other[e / 4][e % 4]));
                    raw[u] = __builtin_bit_cast(i32x4, result);
                }
                uint16_t *const dst = (at[u].kind == QUERY ? q : at[u].kind == KEY ? k : v) + at[u].to + d0;
                if (whole) reinterpret_cast<Loose *>(dst)->v = raw[u];
                else if (held)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (d0 + e < a.dim) dst[e] = (uint16_t)((uint32_t)raw[u][e / 2] >> (e % 2 * 16));
            }
        }
        turn(buffer ^ 1);
        __syncthreads();
    }
}

template <int LANES> void launch_chunks(h3_gpu *g, AxesArgs a) {
    constexpr unsigned GROUPS = 256 / LANES;
    const unsigned items = a.heads + 2 * a.kv_heads;
    // A row's heads go to more workgroups where the rows alone would not fill the chip; rows of few
    // heads share a workgroup's lanes where there are rows enough.
    a.splits = (unsigned)std::min<size_t>((items + GROUPS - 1) / GROUPS, (2048 + (size_t)a.rows - 1) / a.rows);
    a.together = 1;
    while (a.together < TOGETHER && a.splits == 1 && items * a.together * 2 <= 4 * GROUPS && a.rows >= 2 * a.together * 4 * g->cus) a.together *= 2;
    // Many workgroups of a row or few: with as many as run at once the last ones end the call (18,225 rows
    // of 56 heads: 305 us with 4 workgroups a compute unit, 303 with 16, 298 with 64, 291 with one a row).
    const size_t tasks = ((size_t)a.rows + a.together - 1) / a.together * a.splits, each = (tasks + 256 * g->cus - 1) / (256 * g->cus);
    const unsigned blocks = (unsigned)((tasks + each - 1) / each);
    const Pairing pairing = a.interleaved ? NEIGHBOURS : a.dim % 8 == 0 && a.pairs % 8 == 0 ? HALVES : HALVES_LOOSE;
    auto *kernel = pairing == NEIGHBOURS ? rope_axes_chunks<LANES, NEIGHBOURS>
                   : pairing == HALVES   ? rope_axes_chunks<LANES, HALVES>
                                         : rope_axes_chunks<LANES, HALVES_LOOSE>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 2 * a.together * 1024 * sizeof(float), g->compute, a);
}

int rope_axes(h3_gpu *g, const AxesArgs &a) {
    const unsigned chunks = (a.dim + 7) / 8;
    if (chunks <= 2) launch_chunks<2>(g, a);
    else if (chunks <= 4) launch_chunks<4>(g, a);
    else if (chunks <= 8) launch_chunks<8>(g, a);
    else if (chunks <= 16) launch_chunks<16>(g, a);
    else launch_chunks<32>(g, a);
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
                     (const float *)positions->data, rows, heads, kv_heads, heads / kv_heads, dim, rope->pairs,
                     rope->axes, 1, 1, eps, grouped,
                     rope->interleaved};
    return h3_tensors_acquire(g, {qkv, qw, kw, positions}) && rope_axes(g, a) && h3_tensors_release(g, {qkv, qw, kw, positions});
}
