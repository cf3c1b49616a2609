// Block-scaled FP8 matrices (fp8_block.h): their tensors, packing and unpacking, SwiGLU with
// a packed result, and the entry points of the projections and the MLP over them. The norms
// with a packed result are adaln_kernel's (elementwise.hip), the products gemm_fp8_block.hip's.
//
// Packing is one pass, unlike the tensorwide format's (quant.hip): a block's scale needs its
// 128 values only, which eight lanes hold, 16 each.
#include "fp8_block.h"
#include "internal.h"
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// What the context keeps of an MLP's activation.
constexpr size_t MLP_WORKSPACE = (size_t)1 << 30;
constexpr unsigned LANE = 16;                     // values per lane
constexpr unsigned LANES = FP8_BLOCK / LANE;      // lanes per block

// 16 values of a row from `col` on, zeros from `columns` on. VEC: rows of a multiple of eight
// values, so that 16-byte loads are aligned and a half is inside or outside as a whole. Without it
// values are loaded one by one, at a quarter of the rate (SwiGLU of 4000 rows with unpacking: 13824
// wide 83.5 us, 13823 wide 362).
template <bool VEC, class T>
__device__ inline void load16(const T *row, unsigned col, unsigned columns, float *v) {
    constexpr unsigned PER = 16 / sizeof(T);
#pragma unroll
    for (unsigned c = 0; c < LANE; c += PER) {
        if constexpr (VEC) {
            T part[PER] = {};
            if (col + c < columns) *reinterpret_cast<u32x4 *>(part) = *reinterpret_cast<const u32x4 *>(row + col + c);
#pragma unroll
            for (unsigned e = 0; e < PER; e++) {
                if constexpr (sizeof(T) == 2) v[c + e] = bf16_to_f32(part[e]);
                else v[c + e] = part[e];
            }
        } else {
#pragma unroll
            for (unsigned e = 0; e < PER; e++) {
                const T one = col + c + e < columns ? row[col + c + e] : T{};
                if constexpr (sizeof(T) == 2) v[c + e] = bf16_to_f32(one);
                else v[c + e] = one;
            }
        }
    }
}

// The 16 codes of a lane whose block has this scale.
__device__ inline u32x4 encode16(const float *v, unsigned scale) {
    const float value = fp8_block_value(scale);
    return u32x4{fp8_block_encode4(v, value), fp8_block_encode4(v + 4, value), fp8_block_encode4(v + 8, value),
                 fp8_block_encode4(v + 12, value)};
}

// PACK: values of rows [rows, columns]. SWIGLU: silu(gate) * up of rows that hold `columns`
// gate values, then as many up values. Eight lanes per (row, block).
template <bool SWIGLU, bool VEC, class T>
__global__ __launch_bounds__(256) void fp8_block_pack(const T *in, Fp8BlockRows out, unsigned rows, unsigned columns) {
    const unsigned blocks = out.stride / FP8_BLOCK;
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x, item = id / LANES;
    if (item >= (size_t)rows * blocks) return;    // the eight lanes of an item leave together
    const unsigned row = (unsigned)(item / blocks), block = (unsigned)(item % blocks);
    const unsigned col = block * FP8_BLOCK + (unsigned)(id % LANES) * LANE;
    const T *src = in + (size_t)row * columns * (SWIGLU ? 2 : 1);
    float v[LANE];
    if constexpr (!SWIGLU) {
        load16<VEC>(src, col, columns, v);
    } else {
        float gate[LANE], up[LANE];
        load16<VEC>(src, col, columns, gate);
        load16<VEC>(src + columns, col, columns, up);
        swiglu<LANE, false>(gate, up, v);
    }
    bool bad = false;
    const unsigned scale = fp8_block_scale(lanes_max<LANES>(fp8_block_magnitude<LANE>(v, bad)));
    if (bad) *out.fault = 1u;
    *reinterpret_cast<u32x4 *>(out.codes + (size_t)row * out.stride + col) = encode16(v, scale);
    if (id % LANES == 0) out.scales[fp8_block_scale_at(row, block, out.groups)] = (uint8_t)scale;
}

// A weight's blocks of 128 x 128: a workgroup each, 32 rows at a time and eight lanes a row,
// read twice (the second time from L2).
template <bool VEC>
__global__ __launch_bounds__(256) void fp8_block_pack_weight(const uint16_t *in, Fp8BlockRows out, unsigned rows,
                                                             unsigned columns) {
    __shared__ unsigned waves[4];
    const unsigned blocks = out.stride / FP8_BLOCK, block = blockIdx.x % blocks, r0 = blockIdx.x / blocks * FP8_BLOCK;
    const unsigned r = threadIdx.x / LANES, col = block * FP8_BLOCK + threadIdx.x % LANES * LANE;
    unsigned amax = 0;
    bool bad = false;
    float v[LANE];
    for (unsigned at = r; at < FP8_BLOCK && r0 + at < rows; at += 32) {
        load16<VEC>(in + (size_t)(r0 + at) * columns, col, columns, v);
        amax = max(amax, fp8_block_magnitude<LANE>(v, bad));
    }
    if (bad) *out.fault = 1u;
    amax = lanes_max<64>(amax);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = amax;
    __syncthreads();
    const unsigned scale = fp8_block_scale(max(max(waves[0], waves[1]), max(waves[2], waves[3])));
    for (unsigned at = r; at < FP8_BLOCK && r0 + at < rows; at += 32) {
        load16<VEC>(in + (size_t)(r0 + at) * columns, col, columns, v);
        *reinterpret_cast<u32x4 *>(out.codes + (size_t)(r0 + at) * out.stride + col) = encode16(v, scale);
    }
    if (threadIdx.x == 0) out.scales[fp8_block_scale_at(r0 / FP8_BLOCK, block, out.groups)] = (uint8_t)scale;
}

// BF16 values code * 2^e, exact but for values outside BF16's normal range. 16 values per lane.
template <bool VEC>
__global__ __launch_bounds__(256) void fp8_block_unpack(const uint8_t *codes, const uint8_t *scales, unsigned stride,
                                                        unsigned groups, unsigned tile, uint16_t *out,
                                                        unsigned rows, unsigned columns) {
    const unsigned lanes = stride / LANE;
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (size_t)rows * lanes) return;
    const unsigned row = (unsigned)(id / lanes), col = (unsigned)(id % lanes) * LANE;
    if (col >= columns) return;
    const u32x4 q = *reinterpret_cast<const u32x4 *>(codes + (size_t)row * stride + col);
    // Codes times a power of two: exact, and BF16 rounds only what is outside its normal range.
    const int e = (int)scales[fp8_block_scale_at(row / tile, col / FP8_BLOCK, groups)] - 127;
    uint16_t v[LANE];
#pragma unroll
    for (int w = 0; w < 4; w++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f32x2 f = h ? __builtin_amdgcn_cvt_pk_f32_fp8((int)q[w], true)
                              : __builtin_amdgcn_cvt_pk_f32_fp8((int)q[w], false);
            v[4 * w + 2 * h] = f32_to_bf16(__builtin_ldexpf(f[0], e));
            v[4 * w + 2 * h + 1] = f32_to_bf16(__builtin_ldexpf(f[1], e));
        }
    uint16_t *dst = out + (size_t)row * columns + col;
#pragma unroll
    for (unsigned c = 0; c < LANE; c += 8) {
        if constexpr (VEC) {
            if (col + c < columns) *reinterpret_cast<u16x8 *>(dst + c) = *reinterpret_cast<const u16x8 *>(v + c);
        } else {
#pragma unroll
            for (unsigned e = 0; e < 8; e++)
                if (col + c + e < columns) dst[c + e] = v[c + e];
        }
    }
}

constexpr unsigned MAX_GRID = 0x7fffffffu;
// Workgroups of 256 threads, or 0 where they are more than a launch takes.
unsigned grid_of(size_t threads) {
    const size_t groups = (threads + 255) / 256;
    return groups > MAX_GRID / 256 ? 0 : (unsigned)groups;
}

template <bool SWIGLU, class T>
int launch_pack(h3_gpu *g, const T *in, const Fp8BlockRows &out, uint32_t rows, uint32_t columns, const char *what) {
    const unsigned grid = grid_of((size_t)rows * (out.stride / LANE));
    if (!grid) return h3_set_error(g, "%s: %u rows of %u columns are too many for one call", what, rows, columns);
    auto kernel = fp8_block_pack<SWIGLU, true, T>;
    if constexpr (sizeof(T) == 2)           // FP32 rows are the MLP's, a multiple of 128
        if (columns % 8) kernel = fp8_block_pack<SWIGLU, false, T>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, g->compute, in, out, rows, columns);
    return h3_launch_status(g, what);
}

int launch_pack_weight(h3_gpu *g, const uint16_t *in, const Fp8BlockRows &out, uint32_t rows, uint32_t columns) {
    const size_t blocks = (size_t)((rows + FP8_BLOCK - 1) / FP8_BLOCK) * (out.stride / FP8_BLOCK);
    if (!grid_of(blocks * 256)) return h3_set_error(g, "FP8 block weight: %ux%u is too large", rows, columns);
    if (columns % 8 == 0)
        hipLaunchKernelGGL(fp8_block_pack_weight<true>, dim3((unsigned)blocks), dim3(256), 0, g->compute, in, out, rows, columns);
    else
        hipLaunchKernelGGL(fp8_block_pack_weight<false>, dim3((unsigned)blocks), dim3(256), 0, g->compute, in, out, rows, columns);
    return h3_launch_status(g, "FP8 block weight");
}

bool valid_shape(uint32_t rows, uint32_t columns, uint32_t tile) {
    return rows && columns && columns <= FP8_BLOCK_COLUMNS && (tile == 1 || tile == FP8_BLOCK);
}

Fp8BlockLayout layout_of(const h3_gpu_tensor *t) { return fp8_block_layout(t->block_rows, t->block_cols, t->block_tile); }

// Rows of a packed activation over workspace memory (bytes as fp8_block_layout says).
Fp8BlockRows workspace_rows(h3_gpu *g, void *data, uint32_t rows, uint32_t columns) {
    const Fp8BlockLayout l = fp8_block_layout(rows, columns, 1);
    return {(uint8_t *)data, (uint8_t *)data + l.scales, (unsigned)l.stride, (unsigned)l.groups, g->fault + 2};
}

Fp8BlockGemmArgs gemm_args(const h3_gpu_tensor *w, uint32_t rows, uint32_t n) {
    const Fp8BlockLayout lw = layout_of(w);
    Fp8BlockGemmArgs a{};
    a.w = (const uint8_t *)w->data; a.ws = (const uint8_t *)w->data + lw.scales;
    a.m = rows; a.n = n; a.k = (unsigned)lw.stride; a.groups = (unsigned)lw.groups;
    return a;
}

int run_gemm(h3_gpu *g, const h3_gpu_tensor *w, const Fp8BlockGemmArgs &a) {
    if (!h3_tensor_acquire(g, w) || !h3_gemm_fp8_block(g, a)) return 0;
    g->stats.quant_projection_dispatches++;
    g->stats.linear_dispatches++;
    return h3_tensor_release(g, w);
}

// Rows [first, first + m) of a projection; first a multiple of 256: whole runs of 32 scale rows.
Fp8BlockGemmArgs rows_of(Fp8BlockGemmArgs a, uint32_t first, uint32_t m) {
    a.m = m;
    if (a.xb) {
        a.xb += (size_t)first * a.columns;
    } else {
        a.x += (size_t)first * a.k;
        a.xs += fp8_block_scale_at(first, 0, a.groups);
    }
    if (a.y) a.y += (size_t)first * a.n;
    return a;
}

bool overlap(const h3_gpu_tensor *a, const h3_gpu_tensor *b) { return a && b && a->data == b->data; }

}  // namespace

int h3_require_fp8_block(h3_gpu *g, const h3_gpu_tensor *t, uint32_t tile, uint32_t rows, uint32_t columns,
                         const char *name) {
    if (!t) return h3_set_error(g, "%s: missing tensor", name);
    if (t->owner != g) return h3_set_error(g, "%s: tensor belongs to another context", name);
    if (t->block_tile != tile)
        return h3_set_error(g, "%s: need an FP8 block %s", name, tile == 1 ? "activation" : "weight");
    if (t->block_cols != columns || (tile == 1 ? t->block_rows < rows : t->block_rows != rows))
        return h3_set_error(g, "%s: packed matrix is %ux%u, need %ux%u", name, t->block_rows, t->block_cols, rows, columns);
    return 1;
}

Fp8BlockRows h3_fp8_block_rows(h3_gpu *g, const h3_gpu_tensor *t) {
    const Fp8BlockLayout l = layout_of(t);
    return {(uint8_t *)t->data, (uint8_t *)t->data + l.scales, (unsigned)l.stride, (unsigned)l.groups, g->fault + 2};
}

int h3_launch_swiglu_fp8_block(h3_gpu *g, Fp8BlockRows out, const void *fused, bool f32, uint32_t rows, uint32_t width) {
    return f32 ? launch_pack<true>(g, (const float *)fused, out, rows, width, "FP8 block SwiGLU")
               : launch_pack<true>(g, (const uint16_t *)fused, out, rows, width, "FP8 block SwiGLU");
}

// ------------------------------------------------------------------ tensors
extern "C" int h3_hip_fp8_block_layout(uint32_t rows, uint32_t columns, uint32_t tile, size_t *stride, size_t *scales,
                                       size_t *groups, size_t *bytes) {
    if (!valid_shape(rows, columns, tile)) return 0;
    const Fp8BlockLayout l = fp8_block_layout(rows, columns, tile);
    if (stride) *stride = l.stride;
    if (scales) *scales = l.scales;
    if (groups) *groups = l.groups;
    if (bytes) *bytes = l.bytes;
    return 1;
}

extern "C" h3_gpu_tensor *h3_hip_fp8_block_new(h3_gpu *g, uint32_t rows, uint32_t columns, uint32_t tile) {
    if (!g) return nullptr;
    if (!valid_shape(rows, columns, tile)) {
        h3_set_error(g, "FP8 block matrix: %ux%u with tile %u (need rows, 1 to %u columns, tile 1 or 128)", rows, columns,
                     tile, FP8_BLOCK_COLUMNS);
        return nullptr;
    }
    if (h3_capturing(g)) { h3_set_error(g, "FP8 block matrix: the compute stream is being captured"); return nullptr; }
    const Fp8BlockLayout l = fp8_block_layout(rows, columns, tile);
    h3_gpu_tensor *t = h3_gpu_tensor_alloc(g, l.bytes, H3_GPU_I8, H3_GPU_DEVICE_ONLY);
    if (!t) return nullptr;
    t->elements = (size_t)rows * columns;
    t->block_tile = tile; t->block_rows = rows; t->block_cols = columns;
    // Zeros of scale 2^-127; the codes past `columns` stay so.
    if (!h3_hip_check(g, hipMemsetAsync(t->data, 0, l.bytes, g->compute), "FP8 block matrix") ||
        !h3_hip_check(g, hipStreamSynchronize(g->compute), "FP8 block matrix")) {
        h3_gpu_tensor_free(t);
        return nullptr;
    }
    return t;
}

extern "C" h3_gpu_tensor *h3_hip_fp8_block_from_packed(h3_gpu *g, const uint8_t *codes, const uint8_t *scales,
                                                       uint32_t rows, uint32_t columns, uint32_t tile) {
    if (!g) return nullptr;
    if (!codes || !scales) { h3_set_error(g, "FP8 block matrix: missing codes or scales"); return nullptr; }
    if (valid_shape(rows, columns, tile)) {
        const size_t scale_rows = ((size_t)rows + tile - 1) / tile, blocks = (columns + FP8_BLOCK - 1) / FP8_BLOCK;
        if (std::any_of(codes, codes + (size_t)rows * columns, [](uint8_t c) { return (c | 0x80) == 0xff; })) {
            h3_set_error(g, "FP8 block matrix: a code is not a number");
            return nullptr;
        }
        if (std::any_of(scales, scales + scale_rows * blocks, [](uint8_t s) { return s == 0xff; })) {
            h3_set_error(g, "FP8 block matrix: a scale is not a number");
            return nullptr;
        }
        h3_gpu_tensor *t = h3_hip_fp8_block_new(g, rows, columns, tile);
        if (!t) return nullptr;
        const Fp8BlockLayout l = fp8_block_layout(rows, columns, tile);
        std::unique_ptr<uint8_t[]> placed(new (std::nothrow) uint8_t[l.bytes - l.scales]());
        if (!placed) { h3_gpu_tensor_free(t); h3_set_error(g, "FP8 block matrix: out of host memory"); return nullptr; }
        for (uint32_t r = 0; r < scale_rows; r++)
            for (uint32_t b = 0; b < blocks; b++)
                placed[fp8_block_scale_at(r, b, (unsigned)l.groups)] = scales[r * blocks + b];
        if (!h3_hip_check(g, hipMemcpy2D(t->data, l.stride, codes, columns, columns, rows, hipMemcpyHostToDevice),
                          "FP8 block codes upload") ||
            !h3_hip_check(g, hipMemcpy((char *)t->data + l.scales, placed.get(), l.bytes - l.scales, hipMemcpyHostToDevice),
                          "FP8 block scales upload")) {
            h3_gpu_tensor_free(t);
            return nullptr;
        }
        g->stats.h2d_bytes += (size_t)rows * columns + scale_rows * blocks;
        return t;
    }
    return h3_hip_fp8_block_new(g, rows, columns, tile);     // its error
}

extern "C" h3_gpu_tensor *h3_hip_fp8_block_weight_from_bf16(h3_gpu *g, const h3_gpu_tensor *w, uint32_t rows,
                                                            uint32_t columns) {
    if (!g) return nullptr;
    if (!h3_require(g, w, H3_GPU_BF16, (size_t)rows * columns, "FP8 block weight source")) return nullptr;
    h3_gpu_tensor *t = h3_hip_fp8_block_new(g, rows, columns, FP8_BLOCK);
    if (!t) return nullptr;
    // A weight that is not finite is an error here, not at the next submit; a fault that waits for
    // that submit is put aside meanwhile.
    const unsigned none = 0;
    unsigned before = 0, flag = 0, *fault = g->fault + 2;
    int ok = h3_tensor_acquire(g, w) && h3_hip_check(g, hipStreamSynchronize(g->compute), "FP8 block weight") &&
             h3_hip_check(g, hipMemcpy(&before, fault, 4, hipMemcpyDeviceToHost), "FP8 block weight") &&
             (!before || h3_hip_check(g, hipMemcpy(fault, &none, 4, hipMemcpyHostToDevice), "FP8 block weight")) &&
             launch_pack_weight(g, (const uint16_t *)w->data, h3_fp8_block_rows(g, t), rows, columns) &&
             h3_tensor_release(g, w) && h3_hip_check(g, hipStreamSynchronize(g->compute), "FP8 block weight") &&
             h3_hip_check(g, hipMemcpy(&flag, fault, 4, hipMemcpyDeviceToHost), "FP8 block weight");
    if (flag != before)
        ok = h3_hip_check(g, hipMemcpy(fault, &before, 4, hipMemcpyHostToDevice), "FP8 block weight") && ok;
    if (ok && !flag) return t;
    if (ok) h3_set_error(g, "FP8 block weight: nonfinite value");
    h3_gpu_tensor_free(t);
    return nullptr;
}

// ------------------------------------------------------------------ elementwise
extern "C" int h3_hip_fp8_block_pack(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, uint32_t rows,
                                     uint32_t columns) {
    if (!h3_launch_ready(g)) return 0;
    if (!h3_require_fp8_block(g, out, 1, rows, columns, "FP8 block pack output") ||
        !h3_require(g, in, H3_GPU_BF16, (size_t)rows * columns, "FP8 block pack input"))
        return 0;
    return !rows || launch_pack<false>(g, (const uint16_t *)in->data, h3_fp8_block_rows(g, out), rows, columns,
                                       "FP8 block packing");
}

extern "C" int h3_hip_fp8_block_unpack(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, uint32_t rows,
                                       uint32_t columns) {
    if (!h3_launch_ready(g)) return 0;
    if (!in || !in->block_tile) return h3_set_error(g, "FP8 block unpack input: need an FP8 block matrix");
    if (!h3_require_fp8_block(g, in, in->block_tile, rows, columns, "FP8 block unpack input") ||
        !h3_require(g, out, H3_GPU_BF16, (size_t)rows * columns, "FP8 block unpack output"))
        return 0;
    if (!rows) return 1;
    const Fp8BlockLayout l = layout_of(in);
    const unsigned grid = grid_of((size_t)rows * (l.stride / LANE));
    if (!grid) return h3_set_error(g, "FP8 block unpack: %u rows of %u columns are too many for one call", rows, columns);
    auto kernel = columns % 8 == 0 ? fp8_block_unpack<true> : fp8_block_unpack<false>;
    if (!h3_tensor_acquire(g, in)) return 0;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, g->compute, (const uint8_t *)in->data,
                       (const uint8_t *)in->data + l.scales, (unsigned)l.stride, (unsigned)l.groups, in->block_tile,
                       (uint16_t *)out->data, rows, columns);
    return h3_launch_status(g, "FP8 block unpacking") && h3_tensor_release(g, in);
}

extern "C" int h3_hip_swiglu_fp8_block(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *fused, uint32_t rows,
                                       uint32_t width) {
    if (!h3_launch_ready(g)) return 0;
    if (!h3_require_fp8_block(g, out, 1, rows, width, "FP8 block SwiGLU output") ||
        !h3_require(g, fused, H3_GPU_BF16, (size_t)rows * width * 2, "FP8 block SwiGLU input"))
        return 0;
    return !rows || h3_launch_swiglu_fp8_block(g, h3_fp8_block_rows(g, out), fused->data, false, rows, width);
}

// ------------------------------------------------------------------ projections
// The input of a projection (a.m rows of k columns; a's output and weight are set): packed rows
// as they are, a BF16 input packed by the projection itself or here, into the context's
// workspace, whose `extra` bytes behind it *rest is. Refused while the stream is being captured:
// a graph would keep the workspace's address, which later calls use and, growing it, free.
static int projection_input(h3_gpu *g, const h3_gpu_tensor *in, uint32_t k, size_t extra, const char *what,
                            Fp8BlockGemmArgs &a, char **rest) {
    if (in && in->block_tile) {
        if (!h3_require_fp8_block(g, in, 1, a.m, k, what)) return 0;
    } else if (!h3_require(g, in, H3_GPU_BF16, (size_t)a.m * k, what)) {
        return 0;
    }
    const bool pack = !in->block_tile;
    if ((pack || extra) && h3_capturing(g))
        return h3_set_error(g, "%s: needs a workspace, but the compute stream is being captured", what);
    const bool inside = pack && h3_gemm_fp8_block_packs(g, a);
    const size_t own = pack && !inside ? (fp8_block_layout(a.m, k, 1).bytes + 511) & ~(size_t)255 : 0;
    if (own + extra && !h3_buffer_reserve(g, &g->block_workspace, own + extra, what)) return 0;
    *rest = (char *)g->block_workspace.ptr + own;
    if (!h3_tensor_acquire(g, in)) return 0;
    if (inside) {
        a.xb = (const uint16_t *)in->data;
        a.columns = k;
        a.fault = g->fault + 2;
        return 1;
    }
    const Fp8BlockRows x = pack ? workspace_rows(g, g->block_workspace.ptr, a.m, k) : h3_fp8_block_rows(g, in);
    a.x = x.codes;
    a.xs = x.scales;
    return !pack || launch_pack<false>(g, (const uint16_t *)in->data, x, a.m, k, "FP8 block packing");
}

int h3_fp8_block_linear(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w,
                        const h3_gpu_tensor *bias, uint32_t rows, uint32_t k, uint32_t n) {
    if (!h3_launch_ready(g)) return 0;
    if (!rows || !k || !n) return h3_set_error(g, "linear %ux%ux%u: invalid shape", rows, n, k);
    if (!h3_require_fp8_block(g, w, FP8_BLOCK, n, k, "linear weight") ||
        !h3_require(g, out, H3_GPU_BF16, (size_t)rows * n, "linear output") ||
        (bias && !h3_require(g, bias, H3_GPU_BF16, n, "linear bias")))
        return 0;
    if (overlap(out, in) || overlap(out, bias)) return h3_set_error(g, "linear: output aliases input");
    Fp8BlockGemmArgs a = gemm_args(w, rows, n);
    a.y = (uint16_t *)out->data;
    a.bias = bias ? (const uint16_t *)bias->data : nullptr;
    char *rest;
    if (!projection_input(g, in, k, 0, "linear input", a, &rest)) return 0;
    for (uint32_t first = 0; first < rows; first += std::min(rows - first, FP8_BLOCK_ROWS))
        if (!run_gemm(g, w, rows_of(a, first, std::min(rows - first, FP8_BLOCK_ROWS)))) return 0;
    return h3_tensor_release(g, in);
}

int h3_fp8_block_mlp(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w1,
                     const h3_gpu_tensor *w2, uint32_t rows, uint32_t k, uint32_t hidden, uint32_t n) {
    if (!h3_launch_ready(g)) return 0;
    if (h3_capturing(g)) return h3_set_error(g, "MLP: the compute stream is being captured");
    if (!rows || !k || !n || !hidden || hidden % FP8_BLOCK || hidden > FP8_BLOCK_COLUMNS)
        return h3_set_error(g, "MLP %ux%ux%ux%u: need rows, and a hidden width of a multiple of 128 for weights in FP8 "
                               "blocks", rows, k, hidden, n);
    if (!h3_require_fp8_block(g, w1, FP8_BLOCK, 2 * hidden, k, "MLP fc1 weight") ||
        !h3_require_fp8_block(g, w2, FP8_BLOCK, n, hidden, "MLP fc2 weight") ||
        !h3_require(g, out, H3_GPU_BF16, (size_t)rows * n, "MLP output"))
        return 0;
    // The packed activation, and the FP32 product where SwiGLU is not its projection's epilogue.
    // The context keeps no more than MLP_WORKSPACE for them: calls of more rows run in parts.
    const bool fused = h3_gemm_fp8_block_fuses(g, rows, k, hidden);
    const size_t row_bytes = fp8_block_layout(1, hidden, 1).bytes + (fused ? 0 : (size_t)hidden * 8);
    const uint32_t most = (uint32_t)std::min<size_t>(std::max<size_t>(MLP_WORKSPACE / row_bytes / 256, 1) * 256,
                                                     std::min(rows, FP8_BLOCK_ROWS));
    const size_t act = (fp8_block_layout(most, hidden, 1).bytes + 511) & ~(size_t)255;
    Fp8BlockGemmArgs all = gemm_args(w1, rows, 2 * hidden);
    all.swiglu = fused;
    char *rest;
    if (!projection_input(g, in, k, act + (fused ? 0 : (size_t)most * hidden * 8), "MLP input", all, &rest)) return 0;
    // The output may be the input: a BF16 input is packed as a whole first, or by a projection of
    // so few rows that there is one part.
    for (uint32_t first = 0, m; first < rows; first += m) {
        m = std::min(most, rows - first);
        const Fp8BlockRows h = workspace_rows(g, rest, m, hidden);
        Fp8BlockGemmArgs a = rows_of(all, first, m);
        if (fused) a.out = h;
        else a.y32 = (float *)(rest + act);
        if (!run_gemm(g, w1, a) || (!fused && !h3_launch_swiglu_fp8_block(g, h, a.y32, true, m, hidden))) return 0;
        Fp8BlockGemmArgs b = gemm_args(w2, m, n);
        b.x = h.codes;
        b.xs = h.scales;
        b.y = (uint16_t *)out->data + (size_t)first * n;
        if (!run_gemm(g, w2, b)) return 0;
    }
    return h3_tensor_release(g, in);
}

extern "C" int h3_hip_linear_fp8_block(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w,
                                       const h3_gpu_tensor *bias, uint32_t rows, uint32_t k, uint32_t n) {
    if (!h3_launch_ready(g)) return 0;
    if (!in || in->block_tile != 1) return h3_set_error(g, "linear input: need an FP8 block activation");
    return h3_fp8_block_linear(g, out, in, w, bias, rows, k, n);
}

extern "C" int h3_hip_mlp_fp8_block(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w1,
                                    const h3_gpu_tensor *w2, uint32_t rows, uint32_t k, uint32_t hidden, uint32_t n) {
    if (!h3_launch_ready(g)) return 0;
    if (!in || in->block_tile != 1) return h3_set_error(g, "MLP input: need an FP8 block activation");
    return h3_fp8_block_mlp(g, out, in, w1, w2, rows, k, hidden, n);
}
