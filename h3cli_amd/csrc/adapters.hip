// Low-rank adapters of many requests beside a shared projection:
//
//   out[r, :] = base[r, :] + scale_a * (x[r, :] . A_a^T) . B_a^T,     a the adapter of row r
//
// A_a [rank_a, K], B_a [N, rank_a], ranks of their own. Two launches, for all adapters at once:
//  * adapter_down: t = x . A^T in FP32, x read once;
//  * adapter_up: out = base + scale * t . B^T, base read and out written once, whole rows.
// Both are bound by memory: an adapter's flops per byte (rank / 2 of x, rank / 4 of base and out)
// stay far below the matrix cores' share. The plan of the rows (h3_hip_adapter_rows_new) sorts
// them by adapter into tiles of 32, so that a tile has one adapter whatever the rows' order, and
// no tile is larger than a matrix instruction: one row for each of many adapters costs no more
// than their weights' reads.
//
// t enters the second product as two BF16 values, its rounding and what that left: with one,
// the rounding of t would show in the output (2^-9 of the adapter's part), with two its error is
// 2^-18 and the cost a second matrix instruction that memory hides.
#include "common.h"
#include "internal.h"
#include <algorithm>
#include <new>
#include <vector>

struct AdapterEntry {
    uint64_t down, up;     // elements from the start of the packed matrices
    uint32_t blocks;       // 32 ranks each
    float scale;
};

struct h3_hip_adapters {
    h3_gpu *owner;
    uint32_t count, k, n, k_padded;
    std::vector<uint32_t> ranks;
    std::vector<AdapterEntry> entries;
    h3_gpu_tensor *weights;   // BF16: A_a [32 blocks, k_padded] of every adapter, then B_a [n, 32 blocks]
    h3_gpu_tensor *table;     // AdapterEntry [count]
};

struct h3_hip_adapter_rows {
    h3_gpu *owner;
    uint32_t rows, count, max_rank;
    uint32_t tiles, plain;    // tiles of 32 rows with an adapter; behind them those without
    h3_gpu_tensor *order;     // u32 [32 (tiles + plain)]: row, or UINT32_MAX; then the adapter of each tile
    h3_gpu_tensor *sums;      // F32 [splits][32 tiles][padded rank]
    uint32_t splits;          // most K shares of a tile that `sums` holds
};

namespace {

constexpr uint32_t NONE = UINT32_MAX;
constexpr unsigned KC = 64;                // channels of K a step: one cache line of a row
constexpr uint32_t RANK_MOST = 256;

uint32_t rank_blocks(uint32_t rank) { return (rank + 31) / 32; }

struct AdapterArgs {
    uint16_t *out;
    const uint16_t *base, *x;
    const uint16_t *weights;
    const AdapterEntry *table;
    const uint32_t *order, *adapter;       // [32 tiles], [tiles]
    float *sums;
    unsigned rows, count, k, n, k_padded, tiles, passes, splits, rank_padded;
};

// Eight values of a row from channel c on, zeros from `end` on; WIDE: rows start on 16 bytes.
template <bool WIDE> __device__ inline bf16x8 load8(const uint16_t *row, unsigned c, unsigned end) {
    u16x8 v{};
    if constexpr (WIDE) {
        if (c < end) v = *reinterpret_cast<const u16x8 *>(row + c);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (c + e < end) v[e] = row[c + e];
    }
    return __builtin_bit_cast(bf16x8, v);
}

// t of a tile and up to 64 ranks over a share of K: four waves take its 64-channel steps in
// turn and add their sums in LDS, in wave order.
template <bool WIDE>
__global__ __launch_bounds__(256) void adapter_down(AdapterArgs a) {
    __shared__ float part[4][8][64][4];    // [wave][32-rank block * 4 + rows' group][lane]
    const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64, n = lane % 32, hf = lane / 32;
    const unsigned split = blockIdx.x % a.splits, pass = blockIdx.x / a.splits % a.passes, tile = blockIdx.x / a.splits / a.passes;
    const AdapterEntry entry = a.table[a.adapter[tile]];
    if (pass * 2 >= entry.blocks) return;
    const bool both = pass * 2 + 1 < entry.blocks;
    const uint32_t row = a.order[tile * 32 + n];
    const uint16_t *xr = a.x + (size_t)(row == NONE ? a.order[tile * 32] : row) * a.k;
    const uint16_t *down = a.weights + entry.down + (size_t)(pass * 64 + n) * a.k_padded;
    f32x16 acc[2] = {};
    for (unsigned step = split * 4 + wave; step * KC < a.k; step += a.splits * 4) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned c = step * KC + j * 16 + hf * 8;
            const bf16x8 xv = load8<WIDE>(xr, c, a.k);
#pragma unroll
            for (int b = 0; b < 2; b++)
                if (b == 0 || both) {
                    const bf16x8 w = *reinterpret_cast<const bf16x8 *>(down + (size_t)b * 32 * a.k_padded + c);
                    acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, xv, acc[b], 0, 0, 0);
                }
        }
    }
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int q = 0; q < 4; q++)
            *reinterpret_cast<f32x4 *>(part[wave][b * 4 + q][lane]) =
                f32x4{acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
    __syncthreads();
    float *sums = a.sums + ((size_t)(split * a.tiles + tile) * 32 + n) * a.rank_padded + pass * 64;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const unsigned q = wave * 2 + i;   // ranks 32 (q / 4) + 8 (q % 4) + 4 hf + 0..3 of row n
        if (q >= 4 && !both) continue;
        f32x4 t{};
#pragma unroll
        for (int w = 0; w < 4; w++) t += *reinterpret_cast<const f32x4 *>(part[w][q][lane]);
        *reinterpret_cast<f32x4 *>(sums + q / 4 * 32 + q % 4 * 8 + hf * 4) = t;
    }
}

constexpr unsigned COLS = 128;             // columns of a wave's step
constexpr unsigned LDS_ROW = COLS + 4;     // floats: rows of a step shift by four banks

// out = base + scale * t . B^T for a tile's rows and 128 columns a wave; tiles behind the
// adapters' are copied.
template <bool WIDE>
__global__ __launch_bounds__(256) void adapter_up(AdapterArgs a) {
    extern __shared__ __attribute__((aligned(16))) float stage[];
    const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64, n = lane % 32, hf = lane / 32;
    const unsigned groups = (a.n + 4 * COLS - 1) / (4 * COLS);
    const unsigned tile = blockIdx.x / groups, c0 = (blockIdx.x % groups * 4 + wave) * COLS;
    if (c0 >= a.n) return;
    float *const mine = stage + wave * 32 * LDS_ROW;
    const bool adapted = tile < a.tiles;
    if (adapted) {
        const AdapterEntry entry = a.table[a.adapter[tile]];
        const unsigned ranks = entry.blocks * 32;
        f32x16 acc[4] = {};
        for (unsigned r = 0; r < ranks; r += 16) {
            f32x4 t[2] = {};
            for (unsigned split = 0; split < a.splits; split++) {
                const float *p = a.sums + ((size_t)(split * a.tiles + tile) * 32 + n) * a.rank_padded + r + hf * 8;
                t[0] += *reinterpret_cast<const f32x4 *>(p);
                t[1] += *reinterpret_cast<const f32x4 *>(p + 4);
            }
            bf16x8 high, low;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = t[e / 4][e % 4] * entry.scale;
                high[e] = (__bf16)v;
                low[e] = (__bf16)(v - (float)high[e]);
            }
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const unsigned c = min(c0 + b * 32 + n, a.n - 1);
                const bf16x8 w = *reinterpret_cast<const bf16x8 *>(a.weights + entry.up + (size_t)c * ranks + r + hf * 8);
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, high, acc[b], 0, 0, 0);
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, low, acc[b], 0, 0, 0);
            }
        }
        // Row n's columns 32 b + 8 q + 4 hf + 0..3, to be read by whole rows.
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f32x4 *>(mine + n * LDS_ROW + b * 32 + q * 8 + hf * 4) =
                    f32x4{acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own stores
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned r = 4 * i + lane / 16, c = c0 + lane % 16 * 8;
        const uint32_t row = a.order[tile * 32 + r];
        if (row == NONE || c >= a.n) continue;
        const uint16_t *src = a.base + (size_t)row * a.n;
        uint16_t *dst = a.out + (size_t)row * a.n + c;
        u16x8 v = __builtin_bit_cast(u16x8, load8<WIDE>(src, c, a.n));
        if (adapted) {
            const f32x4 d0 = *reinterpret_cast<const f32x4 *>(mine + r * LDS_ROW + lane % 16 * 8);
            const f32x4 d1 = *reinterpret_cast<const f32x4 *>(mine + r * LDS_ROW + lane % 16 * 8 + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = f32_to_bf16(bf16_to_f32(v[e]) + (e < 4 ? d0[e] : d1[e - 4]));
        }
        if constexpr (WIDE) *reinterpret_cast<u16x8 *>(dst) = v;
        else
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (c + e < a.n) dst[e] = v[e];
    }
}

// A [rank, k] into 32 * blocks rows of k_padded values and B [n, rank] into n rows of
// 32 * blocks, zeros behind the ends; without a source (a new adapter) zeros.
__global__ __launch_bounds__(256) void adapter_pack(uint16_t *dst, const uint16_t *src, size_t rows, size_t columns,
                                                    size_t rows_padded, size_t columns_padded) {
    const size_t total = rows_padded * columns_padded;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t r = i / columns_padded, c = i % columns_padded;
        dst[i] = src && r < rows && c < columns ? src[r * columns + c] : (uint16_t)0;
    }
}

void pack(h3_gpu *g, uint16_t *dst, const uint16_t *src, size_t rows, size_t columns, size_t rows_padded, size_t columns_padded) {
    const size_t blocks = std::min<size_t>((rows_padded * columns_padded + 255) / 256, 4096);
    hipLaunchKernelGGL(adapter_pack, dim3((unsigned)blocks), dim3(256), 0, g->compute, dst, src, rows, columns, rows_padded,
                       columns_padded);
}

// Shares of K for `tiles` tiles of up to `passes` * 64 ranks: about two workgroups a compute unit.
uint32_t splits_for(const h3_gpu *g, uint32_t tiles, uint32_t passes) {
    return std::max(1u, std::min(8u, 2 * g->cus / std::max(1u, tiles * passes)));
}

}  // namespace

// ------------------------------------------------------------------ weights
extern "C" void h3_hip_adapters_free(h3_hip_adapters *a) {
    if (!a) return;
    h3_gpu_tensor_free(a->weights);
    h3_gpu_tensor_free(a->table);
    delete a;
}

extern "C" h3_hip_adapters *h3_hip_adapters_new(h3_gpu *g, const uint32_t *ranks, uint32_t count, uint32_t k, uint32_t n) {
    if (!g) return nullptr;
    if (!ranks || !count || count > 65536 || !k || !n || k > (1u << 24) || n > (1u << 24)) {
        h3_set_error(g, "adapters: need 1 to 65536 of them and a projection of up to 2^24 by 2^24");
        return nullptr;
    }
    for (uint32_t i = 0; i < count; i++)
        if (!ranks[i] || ranks[i] > RANK_MOST) {
            h3_set_error(g, "adapters: rank %u of adapter %u, need 1 to %u", ranks[i], i, RANK_MOST);
            return nullptr;
        }
    h3_hip_adapters *a = nullptr;
    size_t elements = 0;
    try {
        a = new h3_hip_adapters{g, count, k, n, (k + KC - 1) / KC * KC, std::vector<uint32_t>(ranks, ranks + count), {}, nullptr, nullptr};
        for (uint32_t i = 0; i < count; i++) {
            const uint64_t blocks = rank_blocks(ranks[i]);
            a->entries.push_back({elements, elements + blocks * 32 * a->k_padded, (uint32_t)blocks, 0.f});
            elements += blocks * 32 * ((size_t)a->k_padded + n);
        }
    } catch (const std::bad_alloc &) {
        delete a;
        h3_set_error(g, "adapters: out of host memory");
        return nullptr;
    }
    a->weights = h3_gpu_tensor_new_bf16(g, elements);
    if (a->weights) {
        pack(g, (uint16_t *)a->weights->data, nullptr, 0, 0, 1, elements);
        a->table = h3_gpu_tensor_from_u32(g, (const uint32_t *)a->entries.data(), count * sizeof(AdapterEntry) / 4);
    }
    if (!a->table || !h3_hip_check(g, hipGetLastError(), "adapters") ||
        !h3_hip_check(g, hipStreamSynchronize(g->compute), "adapters")) {
        h3_hip_adapters_free(a);
        return nullptr;
    }
    return a;
}

__global__ void adapter_entry_scale(AdapterEntry *entry, float scale) { entry->scale = scale; }

extern "C" int h3_hip_adapters_set(h3_gpu *g, h3_hip_adapters *a, uint32_t index, const h3_gpu_tensor *down,
                                   const h3_gpu_tensor *up, float scale) {
    if (!h3_launch_ready(g)) return 0;
    if (!a || a->owner != g || index >= a->count || !finite_f32(scale))
        return h3_set_error(g, "adapters: missing, of another context, index past the last, or a scale that is not finite");
    const uint32_t rank = a->ranks[index];
    if (!h3_require(g, down, H3_GPU_BF16, (size_t)rank * a->k, "adapter A") ||
        !h3_require(g, up, H3_GPU_BF16, (size_t)a->n * rank, "adapter B"))
        return 0;
    AdapterEntry &e = a->entries[index];
    uint16_t *w = (uint16_t *)a->weights->data;
    pack(g, w + e.down, (const uint16_t *)down->data, rank, a->k, (size_t)e.blocks * 32, a->k_padded);
    pack(g, w + e.up, (const uint16_t *)up->data, a->n, rank, a->n, (size_t)e.blocks * 32);
    hipLaunchKernelGGL(adapter_entry_scale, dim3(1), dim3(1), 0, g->compute, (AdapterEntry *)a->table->data + index, scale);
    e.scale = scale;
    return h3_launch_status(g, "adapter");
}

// ------------------------------------------------------------------ rows
extern "C" void h3_hip_adapter_rows_free(h3_hip_adapter_rows *p) {
    if (!p) return;
    h3_gpu_tensor_free(p->order);
    h3_gpu_tensor_free(p->sums);
    delete p;
}

extern "C" h3_hip_adapter_rows *h3_hip_adapter_rows_new(h3_gpu *g, const uint32_t *map, uint32_t rows, uint32_t count,
                                                        uint32_t max_rank) {
    if (!g) return nullptr;
    if (!map || !rows || rows > (1u << 30) || !count || count > 65536 || !max_rank || max_rank > RANK_MOST) {
        h3_set_error(g, "adapter rows: need 1 to 2^30 rows, 1 to 65536 adapters and a rank of 1 to %u", RANK_MOST);
        return nullptr;
    }
    h3_hip_adapter_rows *p = nullptr;
    std::vector<uint32_t> order;
    try {
        p = new h3_hip_adapter_rows{g, rows, count, max_rank, 0, 0, nullptr, nullptr, 1};
        // Rows by adapter, those without (an index past the last) behind them, each in whole tiles.
        std::vector<size_t> start(count + 2, 0);
        for (uint32_t r = 0; r < rows; r++) start[std::min(map[r], count) + 1]++;
        std::vector<uint32_t> adapter;
        for (uint32_t i = 0; i <= count; i++) {
            const size_t tiles = (start[i + 1] + 31) / 32;
            adapter.insert(adapter.end(), tiles, i);
            if (i < count) p->tiles += (uint32_t)tiles;
            else p->plain = (uint32_t)tiles;
            start[i + 1] = start[i] + tiles * 32;
        }
        order.assign(adapter.size() * 32, NONE);
        for (uint32_t r = 0; r < rows; r++) order[start[std::min(map[r], count)]++] = r;
        order.insert(order.end(), adapter.begin(), adapter.end());
    } catch (const std::bad_alloc &) {
        delete p;
        h3_set_error(g, "adapter rows: out of host memory");
        return nullptr;
    }
    const uint32_t blocks = rank_blocks(max_rank);
    p->splits = splits_for(g, p->tiles, (blocks + 1) / 2);
    p->order = h3_gpu_tensor_from_u32(g, order.data(), order.size());
    p->sums = p->order ? h3_gpu_tensor_new_f32(g, std::max<size_t>((size_t)p->splits * p->tiles * 32 * blocks * 32, 1)) : nullptr;
    if (!p->sums) {
        h3_hip_adapter_rows_free(p);
        return nullptr;
    }
    return p;
}

// ------------------------------------------------------------------ operators
static int adapters_valid(h3_gpu *g, const h3_hip_adapters *w, const h3_hip_adapter_rows *p, uint32_t rows, uint32_t k, uint32_t n) {
    if (!w || w->owner != g || !p || p->owner != g)
        return h3_set_error(g, "adapters: missing weights or rows, or of another context");
    if (w->k != k || w->n != n || p->rows != rows || p->count != w->count)
        return h3_set_error(g, "adapters are for %ux%u, %u of them and the rows for %u of %u, need %ux%u and %u rows", w->k, w->n,
                            w->count, p->rows, p->count, k, n, rows);
    for (uint32_t rank : w->ranks)
        if (rank > p->max_rank) return h3_set_error(g, "adapters: rank %u, the rows' plan holds %u", rank, p->max_rank);
    return 1;
}

template <bool WIDE_X, bool WIDE_OUT> static int launch_adapters(h3_gpu *g, const AdapterArgs &a, uint32_t copied) {
    constexpr unsigned shared = 4 * 32 * LDS_ROW * 4;
    static bool configured = false;
    if (!configured) {
        if (!h3_hip_check(g, hipFuncSetAttribute((const void *)adapter_up<WIDE_OUT>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)shared), "adapters' shared memory"))
            return 0;
        configured = true;
    }
    if (a.tiles) {
        hipLaunchKernelGGL(adapter_down<WIDE_X>, dim3(a.tiles * a.passes * a.splits), dim3(256), 0, g->compute, a);
        if (!h3_launch_status(g, "adapters' first product")) return 0;
    }
    const unsigned groups = (a.n + 4 * COLS - 1) / (4 * COLS);
    if (a.tiles + copied)
        hipLaunchKernelGGL(adapter_up<WIDE_OUT>, dim3((a.tiles + copied) * groups), dim3(256), shared, g->compute, a);
    return h3_launch_status(g, "adapters' second product");
}

extern "C" int h3_hip_adapters_add_bf16(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *base, const h3_gpu_tensor *in,
                                        const h3_hip_adapters *w, const h3_hip_adapter_rows *p, uint32_t rows, uint32_t k,
                                        uint32_t n) {
    if (!h3_launch_ready(g) || !adapters_valid(g, w, p, rows, k, n)) return 0;
    if (!h3_require(g, in, H3_GPU_BF16, (size_t)rows * k, "adapters' input") ||
        !h3_require(g, base, H3_GPU_BF16, (size_t)rows * n, "adapters' base") ||
        !h3_require(g, out, H3_GPU_BF16, (size_t)rows * n, "adapters' output"))
        return 0;
    if (out == in) return h3_set_error(g, "adapters: output aliases input");
    uint32_t blocks = 0;
    for (uint32_t rank : w->ranks) blocks = std::max(blocks, rank_blocks(rank));
    const uint32_t groups = (n + 4 * COLS - 1) / (4 * COLS), copied = out->data == base->data ? 0 : p->plain;
    const uint32_t passes = (blocks + 1) / 2, splits = std::min(p->splits, splits_for(g, p->tiles, passes));
    // Launches hold fewer than 2^32 threads.
    if ((uint64_t)(p->tiles + copied) * groups >= (1u << 24) || (uint64_t)p->tiles * passes * splits >= (1u << 24))
        return h3_set_error(g, "adapters: %u rows by %u columns are more than a launch takes", rows, n);
    const AdapterArgs a{(uint16_t *)out->data, (const uint16_t *)base->data, (const uint16_t *)in->data,
                        (const uint16_t *)w->weights->data, (const AdapterEntry *)w->table->data,
                        (const uint32_t *)p->order->data, (const uint32_t *)p->order->data + (size_t)32 * (p->tiles + p->plain),
                        (float *)p->sums->data, rows, w->count, k, n, w->k_padded, p->tiles, passes, splits,
                        rank_blocks(p->max_rank) * 32};
    if (k % 8 == 0) return n % 8 == 0 ? launch_adapters<true, true>(g, a, copied) : launch_adapters<true, false>(g, a, copied);
    return n % 8 == 0 ? launch_adapters<false, true>(g, a, copied) : launch_adapters<false, false>(g, a, copied);
}

extern "C" int h3_hip_linear_adapters_bf16(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *weight,
                                           const h3_gpu_tensor *bias, const h3_hip_adapters *w, const h3_hip_adapter_rows *p,
                                           uint32_t rows, uint32_t k, uint32_t n) {
    return g && h3_launch_ready(g) && adapters_valid(g, w, p, rows, k, n) &&
           h3_gpu_linear_bf16(g, out, in, weight, bias, rows, k, n) &&
           h3_hip_adapters_add_bf16(g, out, out, in, w, p, rows, k, n);
}
