// Low-rank adapters of many requests beside a shared projection:
//
//   out[r, :] = base[r, :] + scale_a * (x[r, :] . A_a^T) . B_a^T,     a the adapter of row r
//
// A_a [rank_a, K], B_a [N, rank_a], ranks of their own. Two launches, for all adapters at once:
//  * adapter_down: t = x . A^T in FP32, x read once for each 64 ranks of the row's adapter;
//  * adapter_up: out = base + scale * t . B^T, base read and out written once, whole rows.
// Both are bound by memory: an adapter's flops per byte (rank / 2 of x, rank / 4 of base and out)
// stay far below the matrix cores' share. The plan of the rows (h3_hip_adapter_rows_new) sorts
// them by adapter into tiles of 32, so that a tile has one adapter whatever the rows' order, and
// no tile is larger than a matrix instruction: one row for each of many adapters costs no more
// than their weights' reads.
//
// t enters the second product as two BF16 values, its rounding and what that left: with one,
// the rounding of t would show in the output (2^-8 of the adapter's part), with two its error is
// 2^-17 and the cost a second matrix instruction that memory hides.
#include "common.h"
#include "internal.h"
#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

struct AdapterEntry {
    uint64_t down, up;     // elements from the start of the packed matrices
    uint32_t rank;
    float scale;
};

struct h3_hip_adapters {
    h3_gpu *owner;
    uint32_t count, k, n, k_padded, n_padded, max_rank;
    std::vector<uint32_t> ranks;
    std::vector<AdapterEntry> entries;
    h3_gpu_tensor *weights;   // BF16: of each A_a, then B_a, as adapter_pack orders them
    h3_gpu_tensor *table;     // AdapterEntry [count]
};

struct h3_hip_adapter_rows {
    h3_gpu *owner;
    uint32_t rows, count, max_rank;
    uint32_t tiles, plain;    // tiles of 32 rows with an adapter; behind them those without
    h3_gpu_tensor *order;     // u32 [32 (tiles + plain)]: row, or UINT32_MAX; then the adapter of each tile
    h3_gpu_tensor *sums;      // F32 [splits][32 tiles][padded rank]
    uint32_t splits;          // most K shares of a tile that `sums` holds
    size_t sums_at;           // behind them adapter_gemm's shared tiles, [SHARED_TILES][64 x 64]
};

namespace {

constexpr uint32_t NONE = UINT32_MAX;
constexpr unsigned KC = 64;                // channels of K a step: one cache line of a row
constexpr unsigned COLS = 64;              // columns of N a step: one cache line of a row
constexpr uint32_t RANK_MOST = 256;
constexpr uint32_t SHARED_TILES = 256;
constexpr uint32_t SPLITS_MOST = 4;   // (eight: 9 rows, 5376 -> 32256, 16.6 us, so 16.0; one: 22)

uint32_t rank_blocks(uint32_t rank) { return (rank + 31) / 32; }

struct AdapterArgs {
    uint16_t *out;
    const uint16_t *base, *x;
    const uint16_t *weights;
    const AdapterEntry *table;
    const uint32_t *order, *adapter;       // [32 tiles], [tiles]
    float *sums;
    const uint16_t *w, *bias;              // adapter_gemm
    float *shared_sums;
    unsigned shares, products;             // and the workgroups of all shares
    unsigned plain;
    unsigned k, n, k_padded, tiles, passes, splits, rank_padded;
    unsigned groups, span;                 // adapter_up: workgroups of a tile, their steps of columns
};

__device__ inline unsigned sixteens_of(const AdapterEntry &e) { return (e.rank + 15) / 16; }

// Ranks `from` to from + 7 of row `row` of t: its shares of K, all on their way at once, and then added
// in order, scaled, and rounded to two BF16 values each: what the first rounding left is in the second
// (nothing where the first is infinite). Ranks that only fill the packed weights up are nothing,
// whatever x holds.
template <unsigned MOST> struct Shares { f32x4 v[MOST][2]; };
template <unsigned MOST> __device__ inline Shares<MOST> shares_of(const AdapterArgs &a, unsigned tile, unsigned row, unsigned from) {
    const float *const p = a.sums + ((size_t)tile * 32 + row) * a.rank_padded + from;
    const size_t stride = (size_t)a.tiles * 32 * a.rank_padded;
    Shares<MOST> s;
#pragma unroll
    for (unsigned split = 0; split < MOST; split++)
        if (MOST == 1 || split < a.splits) {
            s.v[split][0] = *reinterpret_cast<const f32x4 *>(p + split * stride);
            s.v[split][1] = *reinterpret_cast<const f32x4 *>(p + split * stride + 4);
        }
    return s;
}
template <unsigned MOST>
__device__ inline void operands(const AdapterArgs &a, const AdapterEntry &entry, unsigned from, const Shares<MOST> &s, bf16x8 &high,
                                bf16x8 &low) {
    f32x4 t[2] = {};
#pragma unroll
    for (unsigned split = 0; split < MOST; split++)
        if (MOST == 1 || split < a.splits) {
            t[0] += s.v[split][0];
            t[1] += s.v[split][1];
        }
#pragma unroll
    for (unsigned e = 0; e < 8; e++) {
        const float f = from + e < entry.rank ? t[e / 4][e % 4] * entry.scale : 0.f;
        high[e] = (__bf16)f;
        low[e] = (__bf16)(finite_f32((float)high[e]) ? f - (float)high[e] : 0.f);
    }
}

// Eight values from any element on. Global memory takes 16-byte accesses at any two bytes. What lies up
// to 256 bytes behind a tensor's end, more than a step of 64 values, is within its allocation.
struct __attribute__((packed, aligned(2))) Loose { i32x4 v; };
__device__ inline i32x4 load_loose(const uint16_t *p) { return reinterpret_cast<const Loose *>(p)->v; }

// Where chunk c of row r is in LDS, rows of eight 16-byte chunks: sixteen rows' reads of one chunk meet
// sixteen groups of banks.
__device__ inline unsigned swizzled(unsigned r, unsigned c) { return r * 8 + (c ^ r / 2 % 8); }

// The wave's own LDS writes are there, for all its lanes.
__device__ inline void wait_lds() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// t of a tile and up to 64 ranks over a share of K: four waves take its 64-channel steps in turn, the
// next two steps' values of x in flight, and add their sums in LDS, in wave order. x is loaded by
// whole cache lines, eight lanes a row, and goes through 4 KB of LDS a wave (16-byte chunks
// XOR-swizzled) to the lanes that multiply it: loaded as these lanes need it, each line is asked for
// four times, and evicted from the L1 in between.
constexpr unsigned DOWN_WAVES = 4;
__device__ void first_product(const AdapterArgs &a, unsigned id, float *part) {   // part: [wave][32-rank block * 4 + rows' group][lane][4]
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, n = lane % 32, hf = lane / 32;
    const unsigned split = id % a.splits, pass = id / a.splits % a.passes, tile = id / a.splits / a.passes;
    const AdapterEntry entry = a.table[load_uniform(a.adapter + tile)];
    if (pass * 64 >= entry.rank) return;
    const bool both = pass * 64 + 32 < entry.rank;
    // Lane's chunk lane % 8 of rows lane / 8 + 8 i; row r keeps chunk c at swizzled(r, c).
    const unsigned chunk = lane % 8 * 8;
    const uint16_t *xr[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t row = a.order[tile * 32 + lane / 8 + 8 * i];
        if (row == NONE) row = a.order[tile * 32];
        xr[i] = a.x + (size_t)row * a.k + chunk;
    }
    i32x4 *const buffer = reinterpret_cast<i32x4 *>(part + wave * 1024);
    const size_t block_size = (size_t)a.k_padded * 32;
    const uint16_t *const down = a.weights + entry.down + pass * 2 * block_size + lane * 8;
    const unsigned steps = a.k_padded / KC, stride = a.splits * DOWN_WAVES, begin = split * DOWN_WAVES + wave;
    f32x16 acc[2] = {};
    // Loads are made whatever comes of them (behind a row's end, behind the last step): under a
    // condition each would be waited for where it is made.
    auto sum = [&](auto blocks_tag) {
        constexpr int BLOCKS = decltype(blocks_tag)::value;
        i32x4 x[2][4];
        auto load = [&](int slot, unsigned step) {
            step = min(step, steps - 1);
#pragma unroll
            for (int i = 0; i < 4; i++) x[slot][i] = load_loose(xr[i] + step * KC);
        };
        auto multiply = [&](int slot, unsigned step) {
            i32x4 w[BLOCKS][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
                    w[b][j] = *reinterpret_cast<const i32x4 *>(down + b * block_size + (size_t)(step * 4 + j) * 512);
            if (step * KC + KC > a.k)   // what lies behind the row's end is another row's
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (unsigned e = 0; e < 8; e++)
                        if (step * KC + chunk + e >= a.k) x[slot][i][e / 2] &= e % 2 ? 0x0000ffff : 0xffff0000;
            wait_lds();                 // the last step's reads
#pragma unroll
            for (int i = 0; i < 4; i++) buffer[swizzled(lane / 8 + 8 * i, lane % 8)] = x[slot][i];
            wait_lds();
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bf16x8 v = __builtin_bit_cast(bf16x8, buffer[swizzled(n, j * 2 + hf)]);
#pragma unroll
                for (int b = 0; b < BLOCKS; b++)
                    acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w[b][j]), v, acc[b], 0, 0, 0);
            }
        };
        if (begin >= steps) return;
        load(0, begin);
        load(1, begin + stride);
        for (unsigned step = begin; step < steps; step += 2 * stride) {
            multiply(0, step);
            load(0, step + 2 * stride);
            if (step + stride >= steps) break;
            multiply(1, step + stride);
            load(1, step + 3 * stride);
        }
    };
    if (both) sum(std::integral_constant<int, 2>{});
    else sum(std::integral_constant<int, 1>{});
    __syncthreads();                    // the sums take the buffers' place
#pragma unroll
    for (int b = 0; b < 2; b++)
        if (b == 0 || both)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f32x4 *>(part + ((wave * 8 + b * 4 + q) * 64 + lane) * 4) =
                    f32x4{acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
    __syncthreads();
    float *const sums = a.sums + ((size_t)(split * a.tiles + tile) * 32 + n) * a.rank_padded + pass * 64 + hf * 4;
#pragma unroll
    for (unsigned b = 0; b < 2; b++) {
        if (b && !both) break;
        f32x4 t{};
#pragma unroll
        for (unsigned v = 0; v < DOWN_WAVES; v++) t += *reinterpret_cast<const f32x4 *>(part + ((v * 8 + b * 4 + wave) * 64 + lane) * 4);
        *reinterpret_cast<f32x4 *>(sums + b * 32 + wave * 8) = t;     // ranks 32 b + 8 wave + 4 hf + 0..3 of row n
    }
}

__global__ __launch_bounds__(64 * DOWN_WAVES, 2) void adapter_down(AdapterArgs a) {
    extern __shared__ __attribute__((aligned(16))) float part[];
    first_product(a, blockIdx.x, part);
}

constexpr unsigned STAGE_ROW = COLS + 4;   // floats: rows shift by four banks
constexpr unsigned UP_STAGE = 32 * STAGE_ROW;

// out = base + scale * t . B^T for a tile's rows, 64 columns a wave and step; tiles behind the
// adapters' are copied. t is summed over its shares once per workgroup and kept in LDS as the
// two BF16 operands, in the matrix instruction's order. The products go through LDS too, so that base
// and out are read and written by whole cache lines, eight lanes a row. The next weights, and the
// next step's base, are on their way while these are multiplied.
template <bool WIDE>
__global__ __launch_bounds__(256, 2) void adapter_up(AdapterArgs a) {
    extern __shared__ __attribute__((aligned(16))) float shared[];   // [wave] stage, then operands [rank / 16][2][lane]
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, n = lane % 32, hf = lane / 32;
    float *const stage = shared + wave * UP_STAGE;
    i32x4 *const operand = reinterpret_cast<i32x4 *>(shared + 4 * UP_STAGE);
    const unsigned tile = blockIdx.x / a.groups, group = blockIdx.x % a.groups;
    const unsigned steps = (a.n + COLS - 1) / COLS, last = min(steps, (group + 1) * a.span);
    const bool adapted = tile < a.tiles;
    // Lane's chunk lane % 8 of rows lane / 8 + 8 i.
    const unsigned chunk = lane % 8 * 8;
    uint32_t row[4];
#pragma unroll
    for (int i = 0; i < 4; i++) row[i] = a.order[tile * 32 + lane / 8 + 8 * i];
    AdapterEntry entry{};
    if (adapted) entry = a.table[load_uniform(a.adapter + tile)];
    const unsigned sixteens = sixteens_of(entry);
    const uint16_t *const up = a.weights + entry.up + lane * 8;
    i32x4 next_v[4] = {}, next_w[4] = {};
    // Loads are made whatever comes of them (padding rows read row 0, columns behind the end the next
    // row's): under a condition each would be waited for where it is made.
    auto load_base = [&](unsigned step) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint16_t *const p = a.base + (size_t)(row[i] == NONE ? 0 : row[i]) * a.n + step * COLS + chunk;
            if constexpr (WIDE) next_v[i] = *reinterpret_cast<const i32x4 *>(p);
            else next_v[i] = load_loose(p);
        }
    };
    // 32 ranks of the step's 64 columns, the last 16 once more where they end.
    auto load_up = [&](unsigned step, unsigned r) {
#pragma unroll
        for (unsigned i = 0; i < 4; i++)
            next_w[i] = *reinterpret_cast<const i32x4 *>(up + (((size_t)step * sixteens + min(r + i / 2, sixteens - 1)) * 2 + i % 2) * 512);
    };
    unsigned step = group * a.span + wave;
    load_base(min(step, steps - 1));
    if (adapted) {
        load_up(min(step, steps - 1), 0);
        for (unsigned i = threadIdx.x; i < sixteens * 64; i += 256) {
            // Lane i % 64 of rank step i / 64: eight ranks of its row.
            const unsigned from = i / 64 * 16 + i % 64 / 32 * 8;
            bf16x8 high, low;
            operands(a, entry, from, shares_of<SPLITS_MOST>(a, tile, i % 32, from), high, low);
            operand[i / 64 * 128 + i % 64] = __builtin_bit_cast(i32x4, high);
            operand[i / 64 * 128 + 64 + i % 64] = __builtin_bit_cast(i32x4, low);
        }
        __syncthreads();
    }
    for (; step < last; step += 4) {
        i32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = next_v[i];
        const unsigned following = step + 4 < last ? step + 4 : step;   // behind the last one this one, for nothing
        if (adapted) {
            f32x16 acc[2] = {};
            for (unsigned first = 0; first < sixteens; first += 2) {
                i32x4 w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = next_w[i];
                if (first + 2 < sixteens) load_up(step, first + 2);
                else {
                    load_base(following);
                    load_up(following, 0);
                }
#pragma unroll
                for (unsigned r = 0; r < 2; r++) {
                    if (first + r >= sixteens) break;
                    const bf16x8 high = __builtin_bit_cast(bf16x8, operand[(first + r) * 128 + lane]);
                    const bf16x8 low = __builtin_bit_cast(bf16x8, operand[(first + r) * 128 + 64 + lane]);
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const bf16x8 u = __builtin_bit_cast(bf16x8, w[r * 2 + b]);
                        acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u, high, acc[b], 0, 0, 0);
                        acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u, low, acc[b], 0, 0, 0);
                    }
                }
            }
            // Row n's columns 32 b + 8 q + 4 hf + 0..3.
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    *reinterpret_cast<f32x4 *>(stage + n * STAGE_ROW + b * 32 + q * 8 + hf * 4) =
                        f32x4{acc[b][4 * q], acc[b][4 * q + 1], acc[b][4 * q + 2], acc[b][4 * q + 3]};
            wait_lds();
        } else {
            load_base(following);
        }
        const unsigned c = step * COLS + chunk;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (adapted) {
                const f32x4 *const d = reinterpret_cast<const f32x4 *>(stage + (lane / 8 + 8 * i) * STAGE_ROW + chunk);
                const f32x4 d0 = d[0], d1 = d[1];
                bf16x8 y;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t word = (uint32_t)v[i][e / 2];
                    y[e] = (__bf16)(__builtin_bit_cast(float, e % 2 ? word & 0xffff0000u : word << 16) + (e < 4 ? d0[e % 4] : d1[e % 4]));
                }
                v[i] = __builtin_bit_cast(i32x4, y);
            }
            if (row[i] == NONE || c >= a.n) continue;
            uint16_t *const out = a.out + (size_t)row[i] * a.n + c;
            if constexpr (WIDE) __builtin_nontemporal_store(v[i], reinterpret_cast<i32x4 *>(out));
            else if (c + 8 <= a.n) reinterpret_cast<Loose *>(out)->v = v[i];
            else
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c + e < a.n) out[e] = (uint16_t)((uint32_t)v[i][e / 2] >> (e % 2 * 16));
        }
        wait_lds();                     // the stage's reads, before the next step's products
    }
}

// out = x . W^T + bias + the adapters' parts in one sum and one rounding, for BF16 weights whose K is
// no multiple of 64, which the tiled projections do not take. Four waves hold 64 R rows (tiles of
// the rows' plan, so rows of any order) by 64 R columns, 32 R by 32 R each, and go through K
// 64 channels at a time: x and W through two LDS buffers (16-byte chunks XOR-swizzled), the next
// DEPTH steps' values on their way in registers. The adapters' ranks then continue the sum, each row block with
// its adapter's. Bound by the chip's fill at small shapes. At large ones the waves wait for rows that
// pass through registers, since their starts are aligned to two bytes only: 8000 rows, 5001 -> 5001,
// matrix cores and LDS busy for 29% of the time each.
// A compute unit takes in about 20 bytes a cycle of such rows, so few tiles over a long K are shared out
// (part PRODUCT: a share of K, its sums to memory; then part REST: the shares added in order, and
// what follows them). The adapters' first product needs nothing of it and is part of PRODUCT's launch,
// its workgroups behind the shares'. (301 rows, 1001 -> 777: 12.5 us in three shares, unshared, the adapters'
// product before it, 18; 10 rows, 5337 -> 47, 21 shares: 16, 38.)
enum Part { ALL, PRODUCT, REST };
template <int R, Part PART>
__global__ __launch_bounds__(256, 2) void adapter_gemm(AdapterArgs a) {
    constexpr unsigned SIDE = 64 * R, LOADS = SIDE / 32, DEPTH = R == 1 ? 4 : 2;   // LOADS: chunks of each operand a thread
    extern __shared__ __attribute__((aligned(16))) i32x4 lds[];   // [buffer][x, W][SIDE rows of 8 chunks]; then a stage a wave
    const unsigned tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, n = lane % 32, hf = lane / 32;
    if (PART == PRODUCT && blockIdx.x >= a.products) {
        first_product(a, blockIdx.x - a.products, reinterpret_cast<float *>(lds));
        return;
    }
    const unsigned id = PART == PRODUCT ? blockIdx.x / a.shares : blockIdx.x;
    const unsigned tiles_n = (a.n + SIDE - 1) / SIDE, tiles_m = (a.tiles + a.plain + 2 * R - 1) / (2 * R);
    // Columns fastest in bands of eight row tiles, so that what runs together shares both operands.
    const unsigned band = id / (8 * tiles_n), rows_here = min(8u, tiles_m - band * 8), in_band = id - band * 8 * tiles_n;
    const unsigned tm = band * 8 + in_band % rows_here, n0 = in_band / rows_here * SIDE, tile0 = tm * 2 * R;
    const unsigned all = a.tiles + a.plain, chunk = tid % 8 * 8;
    const uint16_t *xr[LOADS], *wr[LOADS];
#pragma unroll
    for (unsigned i = 0; i < LOADS; i++) {
        const unsigned r = tid / 8 + 32 * i, tile = min(tile0 + r / 32, all - 1);
        uint32_t row = a.order[tile * 32 + r % 32];
        if (row == NONE) row = a.order[tile * 32];
        xr[i] = a.x + (size_t)row * a.k + chunk;
        wr[i] = a.w + (size_t)min(n0 + r, a.n - 1) * a.k + chunk;
    }
    i32x4 x[DEPTH][LOADS], w[DEPTH][LOADS];
    const unsigned steps = (a.k + KC - 1) / KC;
    auto load = [&](unsigned slot, unsigned step) {   // behind the last step for nothing
        step = min(step, steps - 1);
#pragma unroll
        for (unsigned i = 0; i < LOADS; i++) {
            x[slot][i] = load_loose(xr[i] + (size_t)step * KC);
            w[slot][i] = load_loose(wr[i] + (size_t)step * KC);
        }
    };
    auto store = [&](unsigned slot, unsigned step) {
        if (step * KC + KC > a.k)       // what lies behind a row's end is another row's
#pragma unroll
            for (unsigned i = 0; i < LOADS; i++)
#pragma unroll
                for (unsigned e = 0; e < 8; e++)
                    if (step * KC + chunk + e >= a.k) {
                        x[slot][i][e / 2] &= e % 2 ? 0x0000ffff : 0xffff0000;
                        w[slot][i][e / 2] &= e % 2 ? 0x0000ffff : 0xffff0000;
                    }
        i32x4 *const to = lds + step % 2 * 2 * SIDE * 8;
#pragma unroll
        for (unsigned i = 0; i < LOADS; i++) {
            const unsigned at = swizzled(tid / 8 + 32 * i, tid % 8);
            to[at] = x[slot][i];
            to[SIDE * 8 + at] = w[slot][i];
        }
    };
    const unsigned wm = wave / 2 * 32 * R, wn = wave % 2 * 32 * R;
    f32x16 acc[R][R] = {};              // [row block][column block]
    if constexpr (PART != REST) {
        const unsigned share = PART == PRODUCT ? blockIdx.x % a.shares : 0;
        const unsigned begin = PART == PRODUCT ? steps * share / a.shares : 0, end = PART == PRODUCT ? steps * (share + 1) / a.shares : steps;
#pragma unroll
        for (unsigned i = 0; i < DEPTH; i++) load(i, begin + i);
        store(0, begin);
        __syncthreads();
        for (unsigned first = begin; first < end; first += DEPTH)
#pragma unroll
        for (unsigned slot = 0; slot < DEPTH; slot++) {
            const unsigned step = first + slot;
            if (step >= end) break;
            load(slot, step + DEPTH);
            const i32x4 *const from = lds + step % 2 * 2 * SIDE * 8;
#pragma unroll
            for (unsigned j = 0; j < 4; j++) {
                bf16x8 xf[R], wf[R];
#pragma unroll
                for (unsigned i = 0; i < R; i++) {
                    xf[i] = __builtin_bit_cast(bf16x8, from[swizzled(wm + 32 * i + n, j * 2 + hf)]);
                    wf[i] = __builtin_bit_cast(bf16x8, from[SIDE * 8 + swizzled(wn + 32 * i + n, j * 2 + hf)]);
                }
#pragma unroll
                for (unsigned i = 0; i < R; i++)
#pragma unroll
                    for (unsigned b = 0; b < R; b++) acc[i][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[b], xf[i], acc[i][b], 0, 0, 0);
            }
            if (step + 1 < end) store((slot + 1) % DEPTH, step + 1);   // last read in the step before this one
            __syncthreads();
        }
    }
    // Shares' sums: [tile][share][wave][register][lane].
    if constexpr (PART == PRODUCT) {
        float *const to = a.shared_sums + ((size_t)blockIdx.x * 4 + wave) * R * R * 16 * 64 + lane;
#pragma unroll
        for (unsigned i = 0; i < R * R * 16; i++) to[i * 64] = acc[i / 16 / R][i / 16 % R][i % 16];
        return;
    }
    if constexpr (PART == REST)
        for (unsigned share0 = 0; share0 < a.shares; share0 += 4) {   // four on their way at a time
            float v[4][R * R * 16];
#pragma unroll
            for (unsigned u = 0; u < 4; u++) {
                const size_t share = (size_t)id * a.shares + min(share0 + u, a.shares - 1);
                const float *const from = a.shared_sums + (share * 4 + wave) * R * R * 16 * 64 + lane;
#pragma unroll
                for (unsigned i = 0; i < R * R * 16; i++) v[u][i] = from[i * 64];
            }
#pragma unroll
            for (unsigned u = 0; u < 4; u++)
                if (share0 + u < a.shares)
#pragma unroll
                    for (unsigned i = 0; i < R * R * 16; i++) acc[i / 16 / R][i / 16 % R][i % 16] += v[u][i];
        }
    float *const stage = reinterpret_cast<float *>(lds) + wave * 32 * (32 * R + 4);
    constexpr unsigned STRIDE = 32 * R + 4, PER_ROW = 4 * R, AT_ONCE = 64 / PER_ROW;   // chunks of a row of the stage
    const unsigned at = lane % PER_ROW * 8, c = n0 + wn + at;
    i32x4 bias{};
    if (a.bias) bias = load_loose(a.bias + (c < a.n ? c : 0));
#pragma unroll
    for (unsigned i = 0; i < R; i++) {
        const unsigned tile = tile0 + wm / 32 + i;
        if (tile >= all) break;
        uint32_t row[32 / AT_ONCE];
#pragma unroll
        for (unsigned j = 0; j < 32 / AT_ONCE; j++) row[j] = a.order[tile * 32 + j * AT_ONCE + lane / PER_ROW];
        if (tile < a.tiles) {
            const AdapterEntry entry = a.table[load_uniform(a.adapter + tile)];
            auto ranks = [&](auto most_tag, auto ahead_tag) {
                constexpr unsigned MOST = decltype(most_tag)::value, AHEAD = decltype(ahead_tag)::value;
                for (unsigned r0 = 0; r0 < entry.rank; r0 += 16 * AHEAD) {
                    Shares<MOST> t[AHEAD];
                    bf16x8 u[AHEAD][R];
#pragma unroll
                    for (unsigned j = 0; j < AHEAD; j++) {
                        const unsigned r = min(r0 + 16 * j, (sixteens_of(entry) - 1) * 16);   // behind the last for nothing
                        t[j] = shares_of<MOST>(a, tile, n, r + hf * 8);
#pragma unroll
                        for (unsigned b = 0; b < R; b++) {
                            // Columns past the last packed step are not stored: any block does.
                            const unsigned c = min(n0 + wn + 32 * b, (a.n - 1) / 32 * 32);
                            u[j][b] = *reinterpret_cast<const bf16x8 *>(
                                a.weights + entry.up + (((size_t)(c / COLS) * sixteens_of(entry) + r / 16) * 2 + c / 32 % 2) * 512 + lane * 8);
                        }
                    }
#pragma unroll
                    for (unsigned j = 0; j < AHEAD; j++) {
                        bf16x8 high, low;
                        operands(a, entry, r0 + 16 * j + hf * 8, t[j], high, low);
#pragma unroll
                        for (unsigned b = 0; b < R; b++) {
                            acc[i][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u[j][b], high, acc[i][b], 0, 0, 0);
                            acc[i][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u[j][b], low, acc[i][b], 0, 0, 0);
                        }
                    }
                }
            };
            if (a.splits == 1) ranks(std::integral_constant<unsigned, 1>{}, std::integral_constant<unsigned, 4>{});
            else ranks(std::integral_constant<unsigned, SPLITS_MOST>{}, std::integral_constant<unsigned, 2>{});
        }
        wait_lds();                     // the stage's last reads
#pragma unroll
        for (unsigned b = 0; b < R; b++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<f32x4 *>(stage + n * STRIDE + b * 32 + q * 8 + hf * 4) =
                    f32x4{acc[i][b][4 * q], acc[i][b][4 * q + 1], acc[i][b][4 * q + 2], acc[i][b][4 * q + 3]};
        wait_lds();
#pragma unroll
        for (unsigned j = 0; j < 32 / AT_ONCE; j++) {
            const unsigned r = j * AT_ONCE + lane / PER_ROW;
            if (row[j] == NONE || c >= a.n) continue;
            bf16x8 y;
#pragma unroll
            for (unsigned e = 0; e < 8; e++) {
                const uint32_t word = (uint32_t)bias[e / 2];
                y[e] = (__bf16)(stage[r * STRIDE + at + e] + __builtin_bit_cast(float, e % 2 ? word & 0xffff0000u : word << 16));
            }
            uint16_t *const out = a.out + (size_t)row[j] * a.n + c;
            const i32x4 v = __builtin_bit_cast(i32x4, y);
            if (c + 8 <= a.n) reinterpret_cast<Loose *>(out)->v = v;
            else
#pragma unroll
                for (unsigned e = 0; e < 8; e++)
                    if (c + e < a.n) out[e] = (uint16_t)((uint32_t)v[e / 2] >> (e % 2 * 16));
        }
    }
}

// A [rank, k] or B [n, rank] in the order in which the kernels' matrix instructions take them, 1 KB each,
// eight values a lane: A's as [32-rank block][16 channels][lane], lane l having rank l % 32 and channels
// 8 (l / 32) on; B's as [64-column step][16 ranks][32 columns of the step][lane], lane l having column
// l % 32 and ranks 8 (l / 32) on. Zeros behind the ends, and without a source (a new adapter).
__global__ __launch_bounds__(256) void adapter_pack(uint16_t *dst, const uint16_t *src, size_t total, size_t rank, size_t other,
                                                    size_t inner, int second) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t e = i % 8, lane = i / 8 % 64, at = i / 512;
        uint16_t v = 0;
        if (!second) {
            const size_t r = at / inner * 32 + lane % 32, k = at % inner * 16 + lane / 32 * 8 + e;
            if (src && r < rank && k < other) v = src[r * other + k];
        } else {
            const size_t c = at / 2 / inner * COLS + at % 2 * 32 + lane % 32;
            const size_t r = at / 2 % inner * 16 + lane / 32 * 8 + e;
            if (src && r < rank && c < other) v = src[c * rank + r];
        }
        dst[i] = v;
    }
}

void pack(h3_gpu *g, uint16_t *dst, const uint16_t *src, size_t total, size_t rank, size_t other, size_t inner, int second) {
    const size_t blocks = std::min<size_t>((total + 255) / 256, 4096);
    hipLaunchKernelGGL(adapter_pack, dim3((unsigned)blocks), dim3(256), 0, g->compute, dst, src, total, rank, other, inner, second);
}

// Shares of K for `tiles` tiles of up to `passes` * 64 ranks: about two workgroups a compute unit.
uint32_t splits_for(const h3_gpu *g, uint32_t tiles, uint32_t passes) {
    return std::max(1u, std::min(SPLITS_MOST, 2 * g->cus / std::max(1u, tiles * passes)));
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
        a = new h3_hip_adapters{g, count, k, n, (k + KC - 1) / KC * KC, (n + COLS - 1) / COLS * COLS,
                                *std::max_element(ranks, ranks + count), std::vector<uint32_t>(ranks, ranks + count), {}, nullptr, nullptr};
        for (uint32_t i = 0; i < count; i++) {
            const size_t down = (size_t)rank_blocks(ranks[i]) * 32 * a->k_padded;
            a->entries.push_back({elements, elements + down, ranks[i], 0.f});
            elements += down + (size_t)((ranks[i] + 15) / 16 * 16) * a->n_padded;
        }
    } catch (const std::bad_alloc &) {
        delete a;
        h3_set_error(g, "adapters: out of host memory");
        return nullptr;
    }
    a->weights = h3_gpu_tensor_new_bf16(g, elements);
    if (a->weights) {
        pack(g, (uint16_t *)a->weights->data, nullptr, elements, 0, 0, 1, 0);
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
    if (!h3_tensors_acquire(g, {down, up})) return 0;
    AdapterEntry &e = a->entries[index];
    uint16_t *w = (uint16_t *)a->weights->data;
    pack(g, w + e.down, (const uint16_t *)down->data, (size_t)rank_blocks(rank) * 32 * a->k_padded, rank, a->k, a->k_padded / 16, 0);
    const uint32_t sixteens = (rank + 15) / 16;
    pack(g, w + e.up, (const uint16_t *)up->data, (size_t)sixteens * 16 * a->n_padded, rank, a->n, sixteens, 1);
    hipLaunchKernelGGL(adapter_entry_scale, dim3(1), dim3(1), 0, g->compute, (AdapterEntry *)a->table->data + index, scale);
    e.scale = scale;
    return h3_launch_status(g, "adapter") && h3_tensors_release(g, {down, up});
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
        p = new h3_hip_adapter_rows{g, rows, count, max_rank, 0, 0, nullptr, nullptr, 1, 0};
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
    p->sums_at = (size_t)p->splits * p->tiles * 32 * blocks * 32;
    p->sums = p->order ? h3_gpu_tensor_new_f32(g, p->sums_at + (size_t)SHARED_TILES * 64 * 64) : nullptr;
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
    if (w->max_rank > p->max_rank) return h3_set_error(g, "adapters: rank %u, the rows' plan holds %u", w->max_rank, p->max_rank);
    return 1;
}

// Launches hold fewer than 2^32 threads.
static int adapters_fit(h3_gpu *g, const h3_hip_adapter_rows *p, uint64_t workgroups, uint32_t rows, uint32_t n) {
    if (workgroups >= (1u << 24) || (uint64_t)p->tiles * ((rank_blocks(p->max_rank) + 1) / 2) * p->splits >= (1u << 24))
        return h3_set_error(g, "adapters: %u rows by %u columns are more than a launch takes", rows, n);
    return 1;
}

static int shared_memory(h3_gpu *g, const void *kernel, size_t bytes) {
    return h3_hip_check(g, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "adapters' shared memory");
}

// The arguments of a call, and its first product.
static int adapters_begin(h3_gpu *g, AdapterArgs &a, const h3_gpu_tensor *in, const h3_hip_adapters *w, const h3_hip_adapter_rows *p,
                          uint32_t &blocks) {
    blocks = rank_blocks(w->max_rank);
    a.x = (const uint16_t *)in->data;
    a.weights = (const uint16_t *)w->weights->data;
    a.table = (const AdapterEntry *)w->table->data;
    a.order = (const uint32_t *)p->order->data;
    a.adapter = a.order + (size_t)32 * (p->tiles + p->plain);
    a.sums = (float *)p->sums->data;
    a.k = w->k;
    a.n = w->n;
    a.k_padded = w->k_padded;
    a.tiles = p->tiles;
    a.plain = p->plain;
    a.passes = (blocks + 1) / 2;
    // No share without a step of 64 channels for each of its waves.
    a.splits = std::min({p->splits, splits_for(g, p->tiles, a.passes), (w->k_padded / KC + DOWN_WAVES - 1) / DOWN_WAVES});
    // Up to 64 steps adapter_gemm takes t in one share, 64 ranks of it on their way at a time, in more shares
    // 32. (301 rows, 2001 -> 777, ranks 16 and 128: 16 us, in eight shares 29; 600 rows, 2001 ->
    // 2001: 41, 61; 10 rows, 5337 -> 47, ranks 16 and 32: 23, 16.)
    if (a.w && w->k_padded / KC <= 64) a.splits = 1;
    a.rank_padded = rank_blocks(p->max_rank) * 32;
    if (!a.tiles || a.products) return 1;   // a shared projection's first launch takes it along
    constexpr unsigned shared = DOWN_WAVES * 8 * 64 * 16;
    static bool configured = false;
    if (!configured && !shared_memory(g, (const void *)adapter_down, shared)) return 0;
    configured = true;
    hipLaunchKernelGGL(adapter_down, dim3(a.tiles * a.passes * a.splits), dim3(64 * DOWN_WAVES), shared, g->compute, a);
    return h3_launch_status(g, "adapters' first product");
}

template <bool WIDE> static int launch_up(h3_gpu *g, const AdapterArgs &a, uint32_t tiles, uint32_t blocks) {
    static bool configured = false;
    if (!configured && !shared_memory(g, (const void *)adapter_up<WIDE>, 4 * UP_STAGE * 4 + RANK_MOST / 32 * 4096)) return 0;
    configured = true;
    hipLaunchKernelGGL(adapter_up<WIDE>, dim3(tiles * a.groups), dim3(256), 4 * UP_STAGE * 4 + blocks * 4096, g->compute, a);
    return h3_launch_status(g, "adapters' second product");
}

template <int R, Part PART> static int launch_gemm(h3_gpu *g, const AdapterArgs &a, uint32_t workgroups) {
    constexpr unsigned shared = 2 * 2 * 64 * R * 128;
    static_assert(4 * 32 * (32 * R + 4) * 4 <= shared, "the stages take the buffers' place");
    static bool configured = false;
    if (!configured && !shared_memory(g, (const void *)adapter_gemm<R, PART>, shared)) return 0;
    configured = true;
    h3_note_kernel(g, "adapter_gemm", 64 * R, a.shares);
    hipLaunchKernelGGL((adapter_gemm<R, PART>), dim3(workgroups), dim3(256), shared, g->compute, a);
    return h3_launch_status(g, "projection with adapters");
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
    const uint32_t tiles = p->tiles + (out->data == base->data ? 0 : p->plain);
    // A workgroup's share of the columns, in steps of 64: few rows in one round of the three
    // workgroups that a compute unit holds, many in four rounds and more.
    const uint32_t steps = (n + COLS - 1) / COLS;
    const uint64_t quads = (uint64_t)tiles * ((steps + 3) / 4), round = 3ull * g->cus;
    AdapterArgs a{};
    a.out = (uint16_t *)out->data;
    a.base = (const uint16_t *)base->data;
    a.span = 4 * (uint32_t)std::min<uint64_t>(8, std::max<uint64_t>(1, quads <= 4 * round ? (quads + round - 1) / round : quads / (4 * round)));
    a.groups = (steps + a.span - 1) / a.span;
    if (!adapters_fit(g, p, (uint64_t)tiles * a.groups, rows, n)) return 0;
    uint32_t blocks;
    if (!h3_tensors_acquire(g, {base, in}) || !adapters_begin(g, a, in, w, p, blocks)) return 0;
    if (tiles && !(n % 8 == 0 ? launch_up<true>(g, a, tiles, blocks) : launch_up<false>(g, a, tiles, blocks))) return 0;
    return h3_tensors_release(g, {base, in});
}

extern "C" int h3_hip_linear_adapters_bf16(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *weight,
                                           const h3_gpu_tensor *bias, const h3_hip_adapters *w, const h3_hip_adapter_rows *p,
                                           uint32_t rows, uint32_t k, uint32_t n) {
    if (!h3_launch_ready(g) || !adapters_valid(g, w, p, rows, k, n)) return 0;
    // The tiled projections take a K of whole 64-channel steps and weights of any type. They write BF16, so
    // that the adapters' parts are added to a rounded sum: one rounding more, 2^-8 of the projection (8193 rows, 7168
    // -> 5376: off by 0.0020 of the result, in one sum 0.0017), for the bits of the projection and
    // h3_hip_adapters_add_bf16 called in turn, whatever the weight's type. Any other K would be gemm_small's, on the
    // vector units, and is adapter_gemm's in one sum. With the adapters: 301 rows, 1001 -> 777: 12.5 us, by
    // gemm_small 140; 8000 rows, 5001 -> 5001: 690-740 us, 541-581 TFLOP/s. Tiles of 64 rows by 64 columns where the large ones would fill few
    // compute units: 600 rows, 2001 -> 3001: 41 us (large 50), 800 rows: 55 (50), 1200 rows, 3001 ->
    // 3001: 93 (65).
    if (!h3_require(g, in, H3_GPU_BF16, (size_t)rows * k, "linear input") ||
        (bias && !h3_require(g, bias, H3_GPU_BF16, n, "linear bias")))
        return 0;
    if (k % KC == 0 || !weight || weight->owner != g || weight->dtype != H3_GPU_BF16 || weight->q8 || weight->quant_mode || weight->block_tile)
        // The projection by itself waits for its weight only, the adapters for x.
        return h3_tensors_acquire(g, {in, bias}) && h3_gpu_linear_bf16(g, out, in, weight, bias, rows, k, n) &&
               h3_hip_adapters_add_bf16(g, out, out, in, w, p, rows, k, n) && h3_tensors_release(g, {bias});
    if (!h3_require(g, weight, H3_GPU_BF16, (size_t)n * k, "linear weight") ||
        !h3_require(g, out, H3_GPU_BF16, (size_t)rows * n, "linear output"))
        return 0;
    if (out == in) return h3_set_error(g, "linear: output aliases input");
    const uint64_t tiles = p->tiles + p->plain;
    const uint64_t large = (tiles + 3) / 4 * ((n + 127) / 128), small = (tiles + 1) / 2 * ((n + 63) / 64);
    if (!adapters_fit(g, p, small, rows, n)) return 0;
    AdapterArgs a{};
    a.out = (uint16_t *)out->data;
    a.w = (const uint16_t *)weight->data;
    a.bias = bias ? (const uint16_t *)bias->data : nullptr;
    a.shared_sums = (float *)p->sums->data + p->sums_at;
    // Four steps of 64 channels a share at least, in one round of the compute units.
    a.shares = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint32_t>(SHARED_TILES, g->cus) / small, (k + KC - 1) / KC / 4));
    a.products = a.shares > 1 ? (uint32_t)small * a.shares : 0;
    uint32_t blocks;
    if (!h3_tensors_acquire(g, {in, weight, bias}) || !adapters_begin(g, a, in, w, p, blocks)) return 0;
    hipEvent_t timing = h3_kernel_timing_begin(g);
    const int ok = a.shares > 1 ? launch_gemm<1, PRODUCT>(g, a, a.products + a.tiles * a.passes * a.splits) &&
                                      launch_gemm<1, REST>(g, a, (uint32_t)small)
                   : large * 5 >= g->cus * 3ull ? launch_gemm<2, ALL>(g, a, (uint32_t)large)
                                                : launch_gemm<1, ALL>(g, a, (uint32_t)small);
    h3_kernel_timing_end(g, timing);
    if (!ok) return 0;
    g->stats.linear_dispatches++;
    return h3_tensors_release(g, {in, weight, bias});
}
