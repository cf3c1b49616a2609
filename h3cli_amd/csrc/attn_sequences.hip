// BF16 attention of packed sequences (D = 128, non-causal): query rows [q0, q0 + lq) of a
// sequence attend to its key rows [k0, k0 + lk), for all sequences in one call
// (h3_hip_sdpa_sequences_bf16). Semantics as attn_bf16.hip: softmax(scale * Q K^T) V with FP32
// scores, running max and sums, P rounded to BF16 for P.V (as the matrix instructions take it: results are
// off by 0.0018 to 0.0023 of their size, of which BF16's own rounding is 0.0017), FP32 accumulation, BF16
// output; a query of a sequence without keys gets zeros.
//
// Query heads that share a key head are rows of one tile: row v of (sequence, key head) is
// query v / share of head share * key head + v % share, so that a key tile is read once for
// all of them and one query of several heads fills more of a matrix instruction.
//
// Three kernels, by how many rows a call has (make_plan):
//  * attn_bf16_pipe (attn_bf16.hip), 256 rows a workgroup, for long sequences: the fastest by row,
//    bound by the matrix cores, but V is transposed first and flagged rows are computed again
//    after it. Four clips of 8193, 301, 2917 and one row, 40 heads: 1.37-1.42 ms, 1.1 PFLOP/s;
//  * attn_sequences_mid, 128 rows, for frames and short clips, one launch. Its matrix and vector
//    instructions take about as long as one another (52 and 50% of the time at 4000 rows) and
//    overlap by two waves a SIMD only. 729 and 806 rows of 56 heads: 54 us;
//  * attn_sequences, 32 rows, its four waves taking the key tiles in turn, for few rows: bound by
//    the keys' reads. Long key ranges go to several workgroups, joined by attn_sequences_join. One to
//    three rows over 18225, 4001, 729 and 9000 keys of 8 key heads (131 MB): 35.5 us, 3.7 TB/s.
#include "common.h"
#include "internal.h"
#include "attn_common.h"
#include <algorithm>
#include <new>
#include <vector>

namespace {

constexpr int D = 128, BN = 64, TILE = BN * D * 2, WAVES = 4;
constexpr float RESCALE_SLACK = 8.0f;
constexpr uint32_t WHOLE = UINT32_MAX, PARTS_MOST = 128;
constexpr uint64_t JOIN_TILES = 8;             // what a join costs, in tiles of a workgroup
constexpr size_t PART_FLOATS = 32 * (D + 2);   // of 32 rows: O, the running max and the sum

// A workgroup's share: 32 rows of a sequence and its key tiles [first, last); part: where its
// partial result goes, WHOLE if it has all tiles. (The sequence is in the item: looked up by its
// index, it would cost a small call one more wait for memory.)
struct RowItem {
    uint32_t q0, lq, k0, lk, block, first, last, part;
};
struct MidItem {
    uint32_t q0, lq, k0, lk, block;   // 128 rows
};
// 32 rows whose tiles were shared out to parts [part, part + parts).
struct JoinItem {
    uint32_t q0, lq, block, part, parts;
};

// What a call does, made on the host.
struct Plan {
    std::vector<h3_sequence> sequences;
    std::vector<h3_sequence_item> tiles, keys;   // by the 256-row tile kernel
    std::vector<MidItem> mid;                    // by attn_sequences_mid
    std::vector<RowItem> rows;                   // by attn_sequences
    std::vector<JoinItem> joins;
    uint64_t vt = 0;                             // elements of transposed V
    uint32_t parts = 0, most_parts = 0;          // in all, and of 32 rows
    size_t table_bytes() const {
        return sequences.size() * sizeof(h3_sequence) + (tiles.size() + keys.size()) * sizeof(h3_sequence_item) +
               mid.size() * sizeof(MidItem) + rows.size() * sizeof(RowItem) + joins.size() * sizeof(JoinItem);
    }
    size_t retry_at() const { return (vt * 2 + 255) / 256 * 256; }
    size_t parts_at(uint32_t kv_heads) const { return (retry_at() + tiles.size() * kv_heads * 8 + 255) / 256 * 256; }
    size_t workspace_bytes(uint32_t kv_heads) const { return parts_at(kv_heads) + (size_t)parts * kv_heads * PART_FLOATS * 4; }
};

}  // namespace

struct h3_hip_sequences {
    h3_gpu *owner;
    uint32_t heads, kv_heads, count;
    uint32_t tiles, keys, mid, rows, joins, most_parts;
    uint64_t q_rows, k_rows;      // rows that the tensors must hold
    size_t retry_at, parts_at;
    h3_gpu_tensor *table;         // h3_sequence, tiles, keys, mid, rows, joins, behind one another
    h3_gpu_tensor *workspace;     // transposed V, retry bytes, partial results
};

namespace {

struct SeqArgs {
    uint16_t *out;
    const uint16_t *q, *k, *v;
    const RowItem *items;
    const MidItem *mid_items;
    const JoinItem *joins;
    float *partial;
    unsigned count, join_count, most_parts, heads, kv_heads, share;
    float scale_log2;
    unsigned *fault;
};

// 16-byte chunk swizzles of a 256-byte row. K: sixteen keys' reads of one chunk meet all banks. V: a
// transposing read takes 32 bytes of each of four keys for 16 lanes, and the 32 bytes behind them for the
// next 16: they meet all banks too. (With K's swizzle for both, 60% of the LDS cycles of the 128-row
// kernel were conflicts: 4000 rows of 40 heads 368 us.)
__device__ inline unsigned chunk(unsigned key, unsigned ch) { return ch ^ (key & 15); }
__device__ inline unsigned v_chunk(unsigned key, unsigned ch) { return ch ^ (key & 3) << 2; }

// The largest exponent field seen, in place (bits 30:23 of a float): non-finite from
// 0x7f800000 on.
__device__ inline void note_bf16(unsigned &worst, const void *values, int words) {
    const uint32_t *w = static_cast<const uint32_t *>(values);
#pragma unroll
    for (int i = 0; i < words; i++) worst = max(max(worst, w[i] & 0x7f800000u), w[i] << 16 & 0x7f800000u);
}

template <int N> __device__ inline void wait_vm_lds() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

typedef short i16x4 __attribute__((ext_vector_type(4)));

// A workgroup of four waves takes 32 rows; its waves take the 64-key tiles in turn, each through
// tiles of its own in LDS (32 KB, no barrier in the loop), and their partial results meet in LDS.
__global__ __attribute__((amdgpu_flat_work_group_size(64 * WAVES, 64 * WAVES), amdgpu_waves_per_eu(2, 2)))
void attn_sequences(SeqArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    __shared__ float mpart[WAVES][32], lpart[WAVES][32];
    const unsigned tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const unsigned n = lane % 32, hf = lane / 32;
    const unsigned id = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned kv = __builtin_amdgcn_readfirstlane(id / a.count);
    const RowItem item = a.items[__builtin_amdgcn_readfirstlane(id % a.count)];
    const unsigned lq = __builtin_amdgcn_readfirstlane(item.lq), lk = __builtin_amdgcn_readfirstlane(item.lk);
    const unsigned q0 = __builtin_amdgcn_readfirstlane(item.q0), k0 = __builtin_amdgcn_readfirstlane(item.k0);
    const unsigned block = __builtin_amdgcn_readfirstlane(item.block);
    const unsigned part = __builtin_amdgcn_readfirstlane(item.part);
    const unsigned rows = lq * a.share, blocks = (rows + 31) / 32, count = __builtin_amdgcn_readfirstlane(item.last);
    const size_t kstride = (size_t)a.kv_heads * D * 2;   // bytes
    const float c = a.scale_log2;
    uint8_t *const kt = smem + wave * 2 * TILE, *const vt = kt + TILE;

    // Tile loads: 1 KB block b of a tile holds keys 4 b + lane / 16, chunk lane % 16 (swizzled).
    // A tile's descriptor starts at its first key and ends with the sequence, or 4 GiB on.
    unsigned off[4], v_off[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned key = 4 * j + lane / 16;
        off[j] = key * (unsigned)kstride + chunk(key, lane % 16) * 16;
        v_off[j] = key * (unsigned)kstride + v_chunk(key, lane % 16) * 16;
    }
    auto load = [&](const uint16_t *base, const unsigned *off, uint8_t *dst, unsigned tile) {
        const unsigned key0 = tile * BN;
        const size_t bytes = (size_t)(lk - key0) * kstride - kv * D * 2;
        const uint16_t *first = base + ((size_t)k0 + key0) * (kstride / 2) + kv * D;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            (void *)first, (short)0, (int)__builtin_amdgcn_readfirstlane((unsigned)(bytes < 0xFFFFFFE0u ? bytes : 0xFFFFFFE0u)), 0x00020000);
        unsigned so = 0;
        const unsigned left = lk - key0 - min(lk - key0, lane / 16);   // keys from this lane's first one on
#pragma unroll 1
        for (int b = 0; b < 16; b += 4) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    r, (__attribute__((address_space(3))) void *)(dst + (b + j) * 1024), 16,
                    left > 4u * (b + j) ? off[j] : BUFFER_OOB, so, 0, 0);
            so = __builtin_amdgcn_readfirstlane(so + 16 * (unsigned)kstride);
        }
    };
    unsigned worst = 0;
    auto screen_tile = [&](const uint8_t *tile) {
#pragma unroll 1
        for (int b = 0; b < 16; b++) {
            const i32x4 w = *reinterpret_cast<const i32x4 *>(tile + (b * 64 + lane) * 16);
            note_bf16(worst, &w, 4);
        }
    };

    // Q fragments (rows past the last repeat it).
    bf16x8 qf[8];
    const unsigned vrow_id = min(block * 32 + n, rows - 1);
    const size_t qrow = ((size_t)q0 + vrow_id / a.share) * a.heads + kv * a.share + vrow_id % a.share;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) qf[ks] = *reinterpret_cast<const bf16x8 *>(a.q + qrow * D + hf * 8 + ks * 16);
    unsigned t = __builtin_amdgcn_readfirstlane(item.first) + wave;
    if (t < count) {
        load(a.k, off, kt, t);
        load(a.v, v_off, vt, t);
    }
    if (wave == 0)
#pragma unroll
        for (int ks = 0; ks < 8; ks++) note_bf16(worst, &qf[ks], 4);
    f32x16 o[4] = {};
    float m = -1e30f, l = 0.f;
    // V^T fragment reads: lane p of a 16-lane group addresses key row p / 4 and channels
    // 4 (p % 4) of a 4 x 16 block and receives channel p of its four keys.
    const unsigned p16 = lane % 16, vrow = hf * 4 + p16 / 4, vch = 2 * (lane / 16 % 2) + p16 % 4 / 2;

    for (; t < count; t += WAVES) {
        const bool more = t + WAVES < count;
        const unsigned key0 = t * BN;
        // Each tile's K and V are screened for Inf and NaN by one of the key head's workgroups.
        const bool screen = t % blocks == block;
        wait_vm_lds<16>();                  // K(t); V(t), loaded after it, may be in flight
        f32x16 sc[2] = {};
        {
            bf16x8 kf[16];
#pragma unroll
            for (int x = 0; x < 16; x++) {
                const unsigned key = x % 2 * 32 + n;
                kf[x] = *reinterpret_cast<const bf16x8 *>(kt + key * 256 + chunk(key, x / 2 * 2 + hf) * 16);
            }
            if (screen) screen_tile(kt);
            wait_vm_lds<16>();              // this wave's reads: the tile may be overwritten
            if (more) load(a.k, off, kt, t + WAVES);
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
#pragma unroll
                for (int mb = 0; mb < 2; mb++)
                    sc[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks * 2 + mb], qf[ks], sc[mb], 0, 0, 0);
        }
        if (key0 + BN > lk)
#pragma unroll
            for (int mb = 0; mb < 2; mb++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (key0 + mb * 32 + (r / 4) * 8 + hf * 4 + r % 4 >= lk) sc[mb][r] = -INFINITY;
        bf16x8 pb[4];
        {
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                mx0 = fmaxf(fmaxf(mx0, sc[0][r]), sc[0][r + 1]);
                mx1 = fmaxf(fmaxf(mx1, sc[1][r]), sc[1][r + 1]);
            }
            const float mx = half_max_swap(fmaxf(mx0, mx1)) * c;
            if (__builtin_amdgcn_ballot_w64(mx > m + RESCALE_SLACK)) {
                const float mnew = fmaxf(m, mx), alpha = exp2f_fast(m - mnew);
                m = mnew;
                l *= alpha;
#pragma unroll
                for (int md = 0; md < 4; md++) o[md] *= alpha;
            }
            const float neg = -m - RESCALE_SLACK;
            float sum = 0.f;
#pragma unroll
            for (int mb = 0; mb < 2; mb++)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float p0 = exp2f_fast(fmaf(sc[mb][r], c, neg)), p1 = exp2f_fast(fmaf(sc[mb][r + 1], c, neg));
                    sum += p0 + p1;
                    pb[mb * 2 + r / 8][r % 8] = (__bf16)p0;
                    pb[mb * 2 + r / 8][r % 8 + 1] = (__bf16)p1;
                }
            l += sum;
        }
        if (more) wait_vm_lds<16>();        // V(t); the next K tile may be in flight
        else wait_vm_lds<0>();
        bf16x8 vf[16];
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
#pragma unroll
            for (int md = 0; md < 4; md++) {
                // Keys 16 kk + 4 hf + 0..3 and 8 further on: the order of P's registers.
                i16x4 half[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned row = 16 * kk + 8 * h + vrow;
                    half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) i16x4 *)(vt + row * 256 + v_chunk(row, md * 4 + vch) * 16 +
                                                                     p16 % 2 * 8));
                }
                vf[kk * 4 + md] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
        if (screen) screen_tile(vt);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) load(a.v, v_off, vt, t + WAVES);
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
#pragma unroll
            for (int md = 0; md < 4; md++)
                o[md] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[kk * 4 + md], pb[kk], o[md], 0, 0, 0);
    }
    wait_vm_loads();

    // The waves' partial results, brought to the common max and added in wave order: wave w
    // finishes channels 32 w .. 32 w + 31.
    if (hf == 0) mpart[wave][n] = m;
    __syncthreads();
    float *const ob = reinterpret_cast<float *>(smem + wave * 2 * TILE);
    {
        float top = mpart[0][n];
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, mpart[w][n]);
        const float alpha = exp2f_fast(m - top), sum = half_sum_swap(l) * alpha;
        if (hf == 0) lpart[wave][n] = sum;
#pragma unroll
        for (int md = 0; md < 4; md++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<f32x4 *>(ob + ((md * 4 + g) * 64 + lane) * 4) =
                    f32x4{o[md][4 * g] * alpha, o[md][4 * g + 1] * alpha, o[md][4 * g + 2] * alpha, o[md][4 * g + 3] * alpha};
    }
    __syncthreads();
    float total = lpart[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; w++) total += lpart[w][n];
    if (part != WHOLE) {
        // The sums over this part's tiles, with their maximum, for attn_sequences_join.
        float *const mine = a.partial + ((size_t)part * a.kv_heads + kv) * PART_FLOATS;
        if (block * 32 + n < rows)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f32x4 x{};
#pragma unroll
                for (int w = 0; w < WAVES; w++)
                    x += *reinterpret_cast<const f32x4 *>(smem + w * 2 * TILE + ((wave * 4 + g) * 64 + lane) * 16);
                *reinterpret_cast<f32x4 *>(mine + n * D + wave * 32 + g * 8 + hf * 4) = x;
            }
        if (wave == 0 && hf == 0) {
            float top = mpart[0][n];
#pragma unroll
            for (int w = 1; w < WAVES; w++) top = fmaxf(top, mpart[w][n]);
            mine[32 * D + n] = top;
            mine[32 * D + 32 + n] = total;
        }
        if (worst >= 0x7f800000u) a.fault[0] = 1u;
        return;
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
    uint16_t *dst = a.out + qrow * D;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        f32x4 x{};
#pragma unroll
        for (int w = 0; w < WAVES; w++)
            x += *reinterpret_cast<const f32x4 *>(smem + w * 2 * TILE + ((wave * 4 + g) * 64 + lane) * 16);
        u16x4 out;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float y = x[e] * inv;
            worst = max(worst, __builtin_bit_cast(uint32_t, y) & 0x7f800000u);
            out[e] = f32_to_bf16(y);
        }
        if (block * 32 + n < rows) *reinterpret_cast<u16x4 *>(dst + wave * 32 + g * 8 + hf * 4) = out;
    }
    if (worst >= 0x7f800000u) a.fault[0] = 1u;
}

// A workgroup of four waves takes 128 rows, 32 a wave, and goes through the key tiles together: each
// tile is loaded once for all waves, the next one on its way in the other of two LDS stages. Two
// workgroups share a compute unit, so that one's softmax runs beside the other's products. Takes the
// sequences that are too short for the 256-row tiles' transposed V and recomputation to pay.
__global__ __attribute__((amdgpu_flat_work_group_size(64 * WAVES, 64 * WAVES), amdgpu_waves_per_eu(2, 2)))
void attn_sequences_mid(SeqArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const unsigned tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const unsigned n = lane % 32, hf = lane / 32;
    const unsigned id = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned kv = __builtin_amdgcn_readfirstlane(id / a.count);
    const MidItem item = a.mid_items[__builtin_amdgcn_readfirstlane(id % a.count)];
    const unsigned lk = __builtin_amdgcn_readfirstlane(item.lk), k0 = __builtin_amdgcn_readfirstlane(item.k0);
    const unsigned block = __builtin_amdgcn_readfirstlane(item.block);
    const unsigned rows = __builtin_amdgcn_readfirstlane(item.lq) * a.share, blocks = (rows + 127) / 128, count = (lk + BN - 1) / BN;
    const size_t kstride = (size_t)a.kv_heads * D * 2;   // bytes
    const float c = a.scale_log2;

    // Wave's 1 KB blocks 4 wave + j of a tile: keys 16 wave + 4 j + lane / 16, chunk lane % 16 (swizzled).
    unsigned off[4], v_off[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned key = 16 * wave + 4 * j + lane / 16;
        off[j] = key * (unsigned)kstride + chunk(key, lane % 16) * 16;
        v_off[j] = key * (unsigned)kstride + v_chunk(key, lane % 16) * 16;
    }
    auto load = [&](const uint16_t *base, const unsigned *off, uint8_t *dst, unsigned tile) {
        const unsigned key0 = tile * BN;
        const size_t bytes = (size_t)(lk - key0) * kstride - kv * D * 2;
        const uint16_t *first = base + ((size_t)k0 + key0) * (kstride / 2) + kv * D;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            (void *)first, (short)0, (int)__builtin_amdgcn_readfirstlane((unsigned)(bytes < 0xFFFFFFE0u ? bytes : 0xFFFFFFE0u)), 0x00020000);
#pragma unroll
        for (unsigned j = 0; j < 4; j++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (__attribute__((address_space(3))) void *)(dst + (wave * 4 + j) * 1024), 16,
                key0 + 16 * wave + 4 * j + lane / 16 < lk ? off[j] : BUFFER_OOB, 0, 0, 0);
    };
    unsigned worst = 0;
    auto screen = [&](const uint8_t *tile) {
#pragma unroll
        for (unsigned j = 0; j < 4; j++) {
            const i32x4 w = *reinterpret_cast<const i32x4 *>(tile + ((wave * 4 + j) * 64 + lane) * 16);
            note_bf16(worst, &w, 4);
        }
    };
    bf16x8 qf[8];
    const unsigned row = block * 128 + wave * 32 + n, held = min(row, rows - 1);
    const size_t qrow = ((size_t)item.q0 + held / a.share) * a.heads + kv * a.share + held % a.share;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) qf[ks] = *reinterpret_cast<const bf16x8 *>(a.q + qrow * D + hf * 8 + ks * 16);
    load(a.k, off, smem, 0);
    load(a.v, v_off, smem + TILE, 0);
#pragma unroll
    for (int ks = 0; ks < 8; ks++) note_bf16(worst, &qf[ks], 4);
    f32x16 o[4] = {};
    float m = -1e30f, l = 0.f;
    const unsigned p16 = lane % 16, vrow = hf * 4 + p16 / 4, vch = 2 * (lane / 16 % 2) + p16 % 4 / 2;
    wait_vm_loads();
    __syncthreads();

    for (unsigned t = 0; t < count; t++) {
        const uint8_t *const kt = smem + t % 2 * 2 * TILE, *const vt = kt + TILE;
        if (t + 1 < count) {
            uint8_t *const next = smem + (t + 1) % 2 * 2 * TILE;
            load(a.k, off, next, t + 1);
            load(a.v, v_off, next + TILE, t + 1);
        }
        // Each tile's K and V are screened for Inf and NaN by one of the key head's workgroups.
        if (t % blocks == block) {
            screen(kt);
            screen(vt);
        }
        f32x16 sc[2] = {};
        {
            bf16x8 kf[16];
#pragma unroll
            for (int x = 0; x < 16; x++) {
                const unsigned key = x % 2 * 32 + n;
                kf[x] = *reinterpret_cast<const bf16x8 *>(kt + key * 256 + chunk(key, x / 2 * 2 + hf) * 16);
            }
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
#pragma unroll
                for (int mb = 0; mb < 2; mb++)
                    sc[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks * 2 + mb], qf[ks], sc[mb], 0, 0, 0);
        }
        // V^T fragments, on their way during the softmax: keys 16 kk + 4 hf + 0..3 and 8 further on, the order
        // of P's registers. (Read after it: 729 and 806 rows of 56 heads 55 us, so 54.)
        i16x4 vh[16][2];
#pragma unroll
        for (int x = 0; x < 16; x++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned r = 16 * (x / 4) + 8 * h + vrow;
                vh[x][h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) i16x4 *)(vt + r * 256 + v_chunk(r, x % 4 * 4 + vch) * 16 + p16 % 2 * 8));
            }
        if (t * BN + BN > lk)
#pragma unroll
            for (int mb = 0; mb < 2; mb++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (t * BN + mb * 32 + (r / 4) * 8 + hf * 4 + r % 4 >= lk) sc[mb][r] = -INFINITY;
        bf16x8 pb[4];
        {
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                mx0 = fmaxf(fmaxf(mx0, sc[0][r]), sc[0][r + 1]);
                mx1 = fmaxf(fmaxf(mx1, sc[1][r]), sc[1][r + 1]);
            }
            const float mx = half_max_swap(fmaxf(mx0, mx1)) * c;
            if (__builtin_amdgcn_ballot_w64(mx > m + RESCALE_SLACK)) {
                const float mnew = fmaxf(m, mx), alpha = exp2f_fast(m - mnew);
                m = mnew;
                l *= alpha;
#pragma unroll
                for (int md = 0; md < 4; md++) o[md] *= alpha;
            }
            const float neg = -m - RESCALE_SLACK;
            float sum = 0.f;
#pragma unroll
            for (int mb = 0; mb < 2; mb++)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float p0 = exp2f_fast(fmaf(sc[mb][r], c, neg)), p1 = exp2f_fast(fmaf(sc[mb][r + 1], c, neg));
                    sum += p0 + p1;
                    pb[mb * 2 + r / 8][r % 8] = (__bf16)p0;
                    pb[mb * 2 + r / 8][r % 8 + 1] = (__bf16)p1;
                }
            l += sum;
        }
#pragma unroll
        for (int x = 0; x < 16; x++) {
            const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(vh[x][0], vh[x][1], 0, 1, 2, 3, 4, 5, 6, 7));
            o[x % 4] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb[x / 4], o[x % 4], 0, 0, 0);
        }
        wait_vm_loads();
        __syncthreads();
    }
    const float total = half_sum_swap(l), inv = total > 0.f ? 1.f / total : 0.f;
    uint16_t *const dst = a.out + qrow * D;
#pragma unroll
    for (int md = 0; md < 4; md++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            u16x4 out;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = o[md][g * 4 + e] * inv;
                worst = max(worst, __builtin_bit_cast(uint32_t, y) & 0x7f800000u);
                out[e] = f32_to_bf16(y);
            }
            if (row < rows) *reinterpret_cast<u16x4 *>(dst + md * 32 + g * 8 + hf * 4) = out;
        }
    if (worst >= 0x7f800000u) a.fault[0] = 1u;
}

// 32 rows from their parts, each brought to the common maximum. JOINERS groups of 256 threads, one or four,
// add every JOINERS-th part, in the parts' order, eight on their way at a time; then the groups' sums
// are added. With the attention, four groups and one: one row of 8 heads over 18225 keys of one head,
// 72 parts, 15.4 and 19.9 us; of 40 heads over 100000 keys of 8, 32 parts, 85.9 and 88.9; ten rows over
// 2000 to 3593 keys, 2 or 3 parts, 34.2 and 33.0.
template <unsigned JOINERS>
__global__ __launch_bounds__(256 * JOINERS) void attn_sequences_join(SeqArgs a) {
    __shared__ float weight[32][PARTS_MOST + 1];
    __shared__ f32x4 sums[JOINERS][256];
    const unsigned tid = threadIdx.x % 256, group = __builtin_amdgcn_readfirstlane(threadIdx.x / 256), kv = blockIdx.x % a.kv_heads;
    const JoinItem item = a.joins[blockIdx.x / a.kv_heads];
    const unsigned rows = min(32u, item.lq * a.share - item.block * 32);
    const float *const first = a.partial + ((size_t)item.part * a.kv_heads + kv) * PART_FLOATS;
    const size_t step = (size_t)a.kv_heads * PART_FLOATS;
    for (unsigned r = threadIdx.x / 32; r < rows; r += 8 * JOINERS) {
        const unsigned lane = threadIdx.x % 32;
        constexpr unsigned EACH = PARTS_MOST / 32;
        float m[EACH], l[EACH], top = -INFINITY, total = 0.f;
#pragma unroll
        for (unsigned i = 0; i < EACH; i++) {   // behind the last part the last again, with no weight
            const float *const at = first + min(lane + 32 * i, item.parts - 1) * step + 32 * D + r;
            m[i] = at[0];
            l[i] = at[32];
        }
#pragma unroll
        for (unsigned i = 0; i < EACH; i++) top = fmaxf(top, m[i]);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
#pragma unroll
        for (unsigned i = 0; i < EACH; i++) {
            const float w = lane + 32 * i < item.parts ? exp2f_fast(m[i] - top) : 0.f;
            weight[r][lane + 32 * i] = w;
            total = fmaf(w, l[i], total);
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
        if (lane == 0) weight[r][PARTS_MOST] = total > 0.f ? 1.f / total : 0.f;
    }
    __syncthreads();
    unsigned worst = 0;
    for (unsigned i0 = 0; i0 < rows * (D / 4); i0 += 256) {
        const unsigned i = i0 + tid, r = min(i / (D / 4), rows - 1), d = i % (D / 4) * 4, v = item.block * 32 + r;
        f32x4 x{};
        for (unsigned p0 = group; p0 < item.parts; p0 += 8 * JOINERS) {
            f32x4 y[8];
#pragma unroll
            for (unsigned p = 0; p < 8; p++)
                y[p] = *reinterpret_cast<const f32x4 *>(first + min(p0 + p * JOINERS, item.parts - 1) * step + r * D + d);
#pragma unroll
            for (unsigned p = 0; p < 8; p++) {
                const bool there = p0 + p * JOINERS < item.parts;
                const float w = there ? weight[r][p0 + p * JOINERS] : 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = there ? fmaf(w, y[p][e], x[e]) : x[e];
            }
        }
        if constexpr (JOINERS > 1) {
            sums[group][tid] = x;
            __syncthreads();
        }
        if (group == 0 && i < rows * (D / 4)) {
#pragma unroll
            for (unsigned j = 1; j < JOINERS; j++) x += sums[j][tid];
            u16x4 out;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = x[e] * weight[r][PARTS_MOST];
                worst = max(worst, __builtin_bit_cast(uint32_t, y) & 0x7f800000u);
                out[e] = f32_to_bf16(y);
            }
            *reinterpret_cast<u16x4 *>(a.out + (((size_t)item.q0 + v / a.share) * a.heads + kv * a.share + v % a.share) * D + d) = out;
        }
        if constexpr (JOINERS > 1) __syncthreads();
    }
    if (worst >= 0x7f800000u) a.fault[0] = 1u;
}

int launch_mid(h3_gpu *g, const SeqArgs &a) {
    constexpr size_t shared = 4 * TILE;
    static bool configured = false;
    if (!configured) {
        if (!h3_hip_check(g, hipFuncSetAttribute((const void *)attn_sequences_mid, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)shared), "attention shared memory"))
            return 0;
        configured = true;
    }
    h3_note_kernel(g, "attn_sequences", 128);
    hipEvent_t timing = h3_kernel_timing_begin(g);
    hipLaunchKernelGGL(attn_sequences_mid, dim3(a.count * a.kv_heads), dim3(64 * WAVES), shared, g->compute, a);
    h3_kernel_timing_end(g, timing);
    return h3_launch_status(g, "BF16 attention of sequences");
}

int launch(h3_gpu *g, const SeqArgs &a) {
    constexpr size_t shared = WAVES * 2 * TILE;
    static bool configured = false;
    if (!configured) {
        if (!h3_hip_check(g, hipFuncSetAttribute((const void *)attn_sequences, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)shared), "attention shared memory"))
            return 0;
        configured = true;
    }
    h3_note_kernel(g, "attn_sequences", 32, a.join_count ? 2 : 1);
    hipEvent_t timing = h3_kernel_timing_begin(g);
    hipLaunchKernelGGL(attn_sequences, dim3(a.count * a.kv_heads), dim3(64 * WAVES), shared, g->compute, a);
    h3_kernel_timing_end(g, timing);
    if (!h3_launch_status(g, "BF16 attention of sequences") || !a.join_count) return h3_launch_status(g, "BF16 attention of sequences");
    if (a.most_parts > 8) hipLaunchKernelGGL(attn_sequences_join<4>, dim3(a.join_count * a.kv_heads), dim3(1024), 0, g->compute, a);
    else hipLaunchKernelGGL(attn_sequences_join<1>, dim3(a.join_count * a.kv_heads), dim3(256), 0, g->compute, a);
    return h3_launch_status(g, "BF16 attention of sequences");
}

// Modelled microseconds of the kernels' workgroups, by 64-key tiles, and of a kernel's launches: as many
// workgroups as run at once, and half a round more behind whole rounds. Measured, all rows by one kernel
// (32 / 128 / 256 rows a workgroup): 300 rows of 4 heads 11 / 13 / 24 us, of 40 heads 19 / 14 / 27;
// 1000 rows of 8 heads 15 / 26 / 34, of 40 heads 62 / 41 / 45; 729 and 806 rows of 56 heads 124 / 56 /
// 76; eight times 250 rows of 40 heads 70 / 29 / 72; 4000 rows of 40 heads 634 / 346 / 332; 5000
// rows of 8 heads 195 / 144 / 118.
struct Load {
    double sum = 0, longest = 0, workgroups = 0;
    void add(double cost, double count) {
        sum += cost * count;
        longest = std::max(longest, cost);
        workgroups += count;
    }
};
double row_cost(uint64_t tiles) { return 6 + 1.75 * (double)((tiles + WAVES - 1) / WAVES); }
double mid_cost(uint64_t tiles) { return 4 + 2.1 * (double)tiles; }              // two on a compute unit
double tile_cost(uint64_t tiles) { return 5 + 2.1 * (double)((tiles + 1) / 2); }
double row_time(const Load &l, double cus) {
    return l.workgroups ? 3 + (l.workgroups > cus ? l.sum / cus + l.longest / 2 : l.longest) : 0;
}
double mid_time(const Load &l, double cus) {
    if (!l.workgroups) return 0;
    return 3 + (l.workgroups > 2 * cus ? l.sum / (2 * cus) + l.longest / 4 : l.workgroups > cus ? l.longest : l.longest * 0.75);
}
// Also the transposition of `keys` keys' V, and the recomputation. Busy compute units draw more power.
double tile_time(const Load &l, double cus, double keys) {
    if (!l.workgroups) return 0;
    return 11 + keys * 1.7e-4 + (1 + 0.45 * std::min(1.0, l.workgroups / cus)) * (l.workgroups > cus ? l.sum / cus + l.longest / 2 : l.longest);
}

// Which kernel takes which sequences, and how the keys of those with few rows are shared out.
const char *make_plan(Plan &plan, const uint32_t *q_offsets, const uint32_t *k_offsets, uint32_t count, uint32_t heads,
                      uint32_t kv_heads, uint32_t cus, int variant) {
    if (!q_offsets || !count || count > (1u << 20) || !kv_heads || !heads || heads > 65535 || heads % kv_heads)
        return "need 1 to 2^20 of them and heads a multiple of the key heads";
    if (!k_offsets) k_offsets = q_offsets;
    const uint32_t share = heads / kv_heads;
    for (uint32_t i = 0; i < count; i++) {
        if (q_offsets[i + 1] < q_offsets[i] || k_offsets[i + 1] < k_offsets[i]) return "the offsets fall";
        const uint64_t lq = q_offsets[i + 1] - q_offsets[i], lk = k_offsets[i + 1] - k_offsets[i];
        if (lq * share >= (1u << 31) || lk >= (1u << 31)) return "a sequence is longer than 2^31 rows";
        plan.sequences.push_back({q_offsets[i], (uint32_t)lq, k_offsets[i], (uint32_t)lk, 0});
    }
    // Those over many keys first within a head's blocks: a short one then ends the head.
    std::vector<uint32_t> order;
    for (uint32_t i = 0; i < count; i++)
        if (plan.sequences[i].lq) order.push_back(i);
    std::stable_sort(order.begin(), order.end(), [&](uint32_t x, uint32_t y) { return plan.sequences[x].lk > plan.sequences[y].lk; });
    auto blocks = [&](uint32_t i, uint32_t size) { return ((uint64_t)plan.sequences[i].lq * share + size - 1) / size; };
    auto tiles = [&](uint32_t i) { return ((uint64_t)plan.sequences[i].lk + BN - 1) / BN; };
    // Kernels in the order of their row blocks: 256, 128 and 32 rows. With the sequences by their rows each
    // kernel takes a range of them; every choice of the two borders (of up to 65 evenly spread ones).
    std::vector<uint32_t> by_rows = order;
    // The tile kernel's offsets into K and into whole tiles of transposed V have 32 bits.
    auto tileable = [&](uint32_t i) { return plan.sequences[i].lk > 256 && tiles(i) * BN * kv_heads * D * 2 < (1ull << 32); };
    std::stable_sort(by_rows.begin(), by_rows.end(), [&](uint32_t x, uint32_t y) { return plan.sequences[x].lq > plan.sequences[y].lq; });
    const size_t n = by_rows.size(), stride = std::max<size_t>(1, (n + 63) / 64);
    // Rows' time from each border on.
    std::vector<size_t> borders;
    for (size_t j = 0; j < n; j += stride) borders.push_back(j);
    borders.push_back(n);
    std::vector<double> rows_from(borders.size(), 0.0);
    Load rows;
    for (size_t b = borders.size() - 1, j = n; b-- > 0;) {
        while (j > borders[b]) {
            j--;
            rows.add(row_cost(tiles(by_rows[j])), (double)blocks(by_rows[j], 32) * kv_heads);
        }
        rows_from[b] = row_time(rows, cus);
    }
    // Sequences above the first border that the tile kernel does not take go to the 128-row kernel, and keep no
    // other from the tiles. (9000 rows over 256 keys beside 8193 over their own, 40 heads: 1363 us; with no tiles
    // for either 1489.)
    double best = 1e300, tile_keys = 0;
    size_t first_mid = 0, first_row = 0, taken = 0;
    Load tile, others;
    for (size_t i = 0; i < borders.size(); i++) {
        for (; taken < borders[i]; taken++) {
            const uint32_t x = by_rows[taken];
            if (!tileable(x)) {
                others.add(mid_cost(tiles(x)), (double)blocks(x, 128) * kv_heads);
                continue;
            }
            tile.add(tile_cost(tiles(x)), (double)blocks(x, 256) * kv_heads);
            tile_keys += (double)plan.sequences[x].lk * kv_heads;
        }
        Load mid = others;
        size_t j = borders[i];
        for (size_t b = i; b < borders.size(); b++) {
            for (; j < borders[b]; j++) mid.add(mid_cost(tiles(by_rows[j])), (double)blocks(by_rows[j], 128) * kv_heads);
            const double time = tile_time(tile, cus, tile_keys) + mid_time(mid, cus) + rows_from[b];
            if (time < best) {
                best = time;
                first_mid = borders[i];
                first_row = j;
            }
        }
    }
    // Measurement: variants 20, 21 and 22 take the kernel of 32 rows, of 128, and of 256 wherever it can.
    if (variant == 20) first_mid = first_row = 0;
    if (variant == 21) first_mid = 0, first_row = n;
    if (variant == 22) first_mid = first_row = n;
    std::vector<uint8_t> kernel(count, 0);
    for (size_t j = 0; j < n; j++) kernel[by_rows[j]] = j < first_mid && tileable(by_rows[j]) ? 2 : j < first_row ? 1 : 0;
    uint64_t work = 0;   // key tiles of the others
    for (uint32_t i : order)
        if (!kernel[i]) work += blocks(i, 32) * kv_heads * tiles(i);
    // A workgroup's share of them: a round of the compute units, each wave with as many tiles as the others.
    // Where that leaves more than a few workgroups for a second round, up to a quarter more, if all then
    // run at once. (Two rows of 56 heads over 9000 keys each: 71 tiles, 224 workgroups, 99 us; 64 tiles, 336
    // workgroups, 128. Rows over 18225, 4001, 729 and 9000 keys of 8 heads: 16 tiles, 264 workgroups,
    // 37 us; 17 tiles, 39.)
    auto parts_of = [&](uint32_t i, uint64_t share) {
        const uint64_t n = tiles(i);
        return n >= share + JOIN_TILES ? std::min<uint64_t>((n + share - 1) / share, PARTS_MOST) : 1;
    };
    auto workgroups = [&](uint64_t share) {
        uint64_t sum = 0;
        for (uint32_t i : order)
            if (!kernel[i]) sum += blocks(i, 32) * kv_heads * parts_of(i, share);
        return sum;
    };
    uint64_t share_tiles = (std::max<uint64_t>(1, (work + cus - 1) / cus) + WAVES - 1) / WAVES * WAVES;
    if (workgroups(share_tiles) > cus + cus / 16)
        for (uint64_t step = 1; step <= 8; step++)
            if (workgroups(share_tiles + share_tiles * step / 32) <= cus) {
                share_tiles += share_tiles * step / 32;
                break;
            }
    for (uint32_t i : order) {
        h3_sequence &s = plan.sequences[i];
        // Launches hold fewer than 2^32 threads.
        if (kernel[i] == 1) {
            if ((plan.mid.size() + blocks(i, 128)) * kv_heads >= (1u << 24)) return "more rows than a launch takes";
            for (uint32_t b = 0; b < blocks(i, 128); b++) plan.mid.push_back({s.q0, s.lq, s.k0, s.lk, b});
            continue;
        }
        if (kernel[i] == 2) {
            if ((plan.tiles.size() + blocks(i, 256)) * kv_heads >= (1u << 23) || (plan.keys.size() + tiles(i)) * kv_heads >= (1u << 24))
                return "more rows than a launch takes";
            s.vt = plan.vt;
            plan.vt += (uint64_t)tiles(i) * BN * D * kv_heads;
            for (uint32_t b = 0; b < blocks(i, 256); b++) plan.tiles.push_back({i, b});
            for (uint32_t b = 0; b < tiles(i); b++) plan.keys.push_back({i, b});
            continue;
        }
        const uint64_t n = tiles(i), parts = parts_of(i, share_tiles);
        if ((plan.rows.size() + blocks(i, 32) * parts) * kv_heads >= (1u << 24)) return "more rows than a launch takes";
        plan.most_parts = std::max(plan.most_parts, (uint32_t)parts);
        for (uint32_t b = 0; b < blocks(i, 32); b++) {
            if (parts > 1) plan.joins.push_back({s.q0, s.lq, b, plan.parts, (uint32_t)parts});
            for (uint64_t p = 0; p < parts; p++)
                plan.rows.push_back({s.q0, s.lq, s.k0, s.lk, b, (uint32_t)(n * p / parts), (uint32_t)(n * (p + 1) / parts),
                                     parts > 1 ? plan.parts++ : WHOLE});
        }
    }
    return nullptr;
}

}  // namespace

extern "C" void h3_hip_sequences_free(h3_hip_sequences *s) {
    if (!s) return;
    h3_gpu_tensor_free(s->table);
    h3_gpu_tensor_free(s->workspace);
    delete s;
}

extern "C" int h3_hip_sequences_layout(const uint32_t *q_offsets, const uint32_t *k_offsets, uint32_t count, uint32_t heads,
                                       uint32_t kv_heads, size_t *bytes) try {
    Plan plan;
    if (make_plan(plan, q_offsets, k_offsets, count, heads, kv_heads, 256, 0)) return 0;
    if (bytes) *bytes = plan.table_bytes() + plan.workspace_bytes(kv_heads);
    return 1;
} catch (const std::bad_alloc &) {
    return 0;
}

extern "C" h3_hip_sequences *h3_hip_sequences_new(h3_gpu *g, const uint32_t *q_offsets, const uint32_t *k_offsets, uint32_t count,
                                                  uint32_t heads, uint32_t kv_heads) {
    if (!g) return nullptr;
    h3_hip_sequences *s = nullptr;
    Plan plan;
    std::vector<uint32_t> words;
    try {
        if (const char *why = make_plan(plan, q_offsets, k_offsets, count, heads, kv_heads, g->cus, g->attention_variant)) {
            h3_set_error(g, "sequences: %s", why);
            return nullptr;
        }
        auto append = [&](const auto &list) {
            const auto *w = reinterpret_cast<const uint32_t *>(list.data());
            words.insert(words.end(), w, w + list.size() * sizeof(list[0]) / 4);
        };
        append(plan.sequences);
        append(plan.tiles);
        append(plan.keys);
        append(plan.mid);
        append(plan.rows);
        append(plan.joins);
        s = new h3_hip_sequences{g, heads, kv_heads, count, (uint32_t)plan.tiles.size(), (uint32_t)plan.keys.size(),
                                 (uint32_t)plan.mid.size(), (uint32_t)plan.rows.size(), (uint32_t)plan.joins.size(),
                                 plan.most_parts, q_offsets[count],
                                 (k_offsets ? k_offsets : q_offsets)[count], plan.retry_at(), plan.parts_at(kv_heads), nullptr, nullptr};
    } catch (const std::bad_alloc &) {
        h3_set_error(g, "sequences: out of host memory");
        return nullptr;
    }
    s->table = h3_gpu_tensor_from_u32(g, words.data(), words.size());
    if (s->table && plan.workspace_bytes(kv_heads))
        s->workspace = h3_gpu_tensor_alloc(g, plan.workspace_bytes(kv_heads), H3_GPU_I8, H3_GPU_DEVICE_ONLY);
    if (!s->table || (plan.workspace_bytes(kv_heads) && !s->workspace)) {
        h3_hip_sequences_free(s);
        return nullptr;
    }
    return s;
}

extern "C" int h3_hip_sdpa_sequences_bf16(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *q, const h3_gpu_tensor *k,
                                          const h3_gpu_tensor *v, const h3_hip_sequences *s, float scale) {
    if (!h3_launch_ready(g)) return 0;
    if (!s || s->owner != g) return h3_set_error(g, "attention of sequences: missing plan, or of another context");
    if (!finite_f32(scale) || scale <= 0 || !out || out == q || out == k || out == v)
        return h3_set_error(g, "attention of sequences requires a disjoint BF16 output and a positive FP32 scale");
    const size_t nq = (size_t)s->q_rows * s->heads * D, nk = (size_t)s->k_rows * s->kv_heads * D;
    if (!h3_require(g, q, H3_GPU_BF16, nq, "attention Q") || !h3_require(g, k, H3_GPU_BF16, nk, "attention K") ||
        !h3_require(g, v, H3_GPU_BF16, nk, "attention V") || !h3_require(g, out, H3_GPU_BF16, nq, "attention output"))
        return 0;
    const float rounded = bf16_to_f32(f32_to_bf16(scale));
    const auto *sequences = (const h3_sequence *)s->table->data;
    const auto *items = (const h3_sequence_item *)(sequences + s->count);
    const auto *mid = (const MidItem *)(items + s->tiles + s->keys);
    const auto *rows = (const RowItem *)(mid + s->mid);
    char *const workspace = s->workspace ? (char *)s->workspace->data : nullptr;
    if (!h3_tensors_acquire(g, {q, k, v})) return 0;
    if (s->tiles) {
        const h3_sequence_tiles t{sequences, items, items + s->tiles, s->tiles, s->keys, s->heads, s->kv_heads,
                                  (uint16_t *)workspace, (uint8_t *)workspace + s->retry_at};
        if (!h3_launch_attention_sequence_tiles(g, (uint16_t *)out->data, (const uint16_t *)q->data, (const uint16_t *)k->data,
                                                (const uint16_t *)v->data, t, rounded))
            return 0;
    }
    SeqArgs a{(uint16_t *)out->data, (const uint16_t *)q->data, (const uint16_t *)k->data, (const uint16_t *)v->data, rows, mid,
              (const JoinItem *)(rows + s->rows), s->joins ? (float *)(workspace + s->parts_at) : nullptr,
              s->mid, s->joins, s->most_parts, s->heads, s->kv_heads, s->heads / s->kv_heads, rounded * 1.4426950408889634f, g->fault};
    if (s->mid && !launch_mid(g, a)) return 0;
    a.count = s->rows;
    if (s->rows && !launch(g, a)) return 0;
    if (s->tiles + s->mid + s->rows) g->stats.attention_dispatches++;
    return h3_tensors_release(g, {q, k, v});
}
