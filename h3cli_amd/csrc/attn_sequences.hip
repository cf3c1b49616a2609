// BF16 attention of packed sequences (D = 128, non-causal): query rows [q0, q0 + lq) of a
// sequence attend to its key rows [k0, k0 + lk), for all sequences in one call
// (h3_hip_sdpa_sequences_bf16). Semantics as attn_bf16.hip: softmax(scale * Q K^T) V with FP32
// scores, running max and sums, P rounded to BF16 for P.V, FP32 accumulation, BF16 output; a
// query of a sequence without keys gets zeros.
//
// Query heads that share a key head are rows of one tile: row v of (sequence, key head) is
// query v / share of head share * key head + v % share, so that a key tile is read once for
// all of them and one query of several heads fills more of a matrix instruction.
#include "common.h"
#include "internal.h"
#include "attn_common.h"
#include <algorithm>
#include <new>
#include <vector>

namespace {

constexpr int D = 128, BN = 64, TILE = BN * D * 2, WAVES = 4;
constexpr float RESCALE_SLACK = 8.0f;

struct Sequence {
    uint32_t q0, lq, k0, lk;
};
// A workgroup's share: a block of rows of a sequence.
struct Item {
    uint32_t sequence, block;
};

}  // namespace

struct h3_hip_sequences {
    h3_gpu *owner;
    uint32_t heads, kv_heads, count, items;
    uint64_t q_rows, k_rows;      // rows that the tensors must hold
    h3_gpu_tensor *table;         // u32: Sequence [count], Item [items]
};

namespace {

struct SeqArgs {
    uint16_t *out;
    const uint16_t *q, *k, *v;
    const Sequence *sequences;
    const Item *items;
    unsigned count, heads, kv_heads, share;
    float scale_log2;
    unsigned *fault;
};

// 16-byte chunk swizzle of a 256-byte row.
__device__ inline unsigned chunk(unsigned key, unsigned ch) { return ch ^ (key & 15); }

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
    const Item item = a.items[__builtin_amdgcn_readfirstlane(id % a.count)];
    const Sequence s = a.sequences[item.sequence];
    const unsigned lq = __builtin_amdgcn_readfirstlane(s.lq), lk = __builtin_amdgcn_readfirstlane(s.lk);
    const unsigned q0 = __builtin_amdgcn_readfirstlane(s.q0), k0 = __builtin_amdgcn_readfirstlane(s.k0);
    const unsigned block = __builtin_amdgcn_readfirstlane(item.block);
    const unsigned rows = lq * a.share, blocks = (rows + 31) / 32, count = (lk + BN - 1) / BN;
    const size_t kstride = (size_t)a.kv_heads * D * 2;   // bytes
    const float c = a.scale_log2;
    uint8_t *const kt = smem + wave * 2 * TILE, *const vt = kt + TILE;

    // Tile loads: 1 KB block b of a tile holds keys 4 b + lane / 16, chunk lane % 16 (swizzled).
    // A tile's descriptor starts at its first key and ends with the sequence, or 4 GiB on.
    unsigned off[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned key = 4 * j + lane / 16;
        off[j] = key * (unsigned)kstride + chunk(key, lane % 16) * 16;
    }
    auto load = [&](const uint16_t *base, uint8_t *dst, unsigned tile) {
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
    unsigned t = wave;
    if (t < count) {
        load(a.k, kt, t);
        load(a.v, vt, t);
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
            if (more) load(a.k, kt, t + WAVES);
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
                        (__attribute__((address_space(3))) i16x4 *)(vt + row * 256 + chunk(row, md * 4 + vch) * 16 +
                                                                     p16 % 2 * 8));
                }
                vf[kk * 4 + md] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
        if (screen) screen_tile(vt);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) load(a.v, vt, t + WAVES);
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

int launch(h3_gpu *g, const SeqArgs &a) {
    constexpr size_t shared = WAVES * 2 * TILE;
    static bool configured = false;
    if (!configured) {
        if (!h3_hip_check(g, hipFuncSetAttribute((const void *)attn_sequences, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)shared), "attention shared memory"))
            return 0;
        configured = true;
    }
    h3_note_kernel(g, "attn_sequences");
    hipEvent_t timing = h3_kernel_timing_begin(g);
    hipLaunchKernelGGL(attn_sequences, dim3(a.count * a.kv_heads), dim3(64 * WAVES), shared, g->compute, a);
    h3_kernel_timing_end(g, timing);
    return h3_launch_status(g, "BF16 attention of sequences");
}

}  // namespace

extern "C" void h3_hip_sequences_free(h3_hip_sequences *s) {
    if (!s) return;
    h3_gpu_tensor_free(s->table);
    delete s;
}

extern "C" h3_hip_sequences *h3_hip_sequences_new(h3_gpu *g, const uint32_t *q_offsets, const uint32_t *k_offsets, uint32_t count,
                                                  uint32_t heads, uint32_t kv_heads) {
    if (!g) return nullptr;
    if (!q_offsets || !count || count > (1u << 20) || !kv_heads || !heads || heads > 65535 || heads % kv_heads) {
        h3_set_error(g, "sequences: need 1 to 2^20 of them and heads a multiple of the key heads");
        return nullptr;
    }
    if (!k_offsets) k_offsets = q_offsets;
    const uint32_t share = heads / kv_heads;
    h3_hip_sequences *s = nullptr;
    std::vector<uint32_t> words;
    try {
        std::vector<Item> items;
        for (uint32_t i = 0; i < count; i++) {
            if (q_offsets[i + 1] < q_offsets[i] || k_offsets[i + 1] < k_offsets[i]) {
                h3_set_error(g, "sequences: offsets of sequence %u fall", i);
                return nullptr;
            }
            const uint64_t lq = q_offsets[i + 1] - q_offsets[i], lk = k_offsets[i + 1] - k_offsets[i];
            if (lq * share >= (1u << 31) || lk >= (1u << 31)) {
                h3_set_error(g, "sequences: sequence %u is longer than 2^31 rows", i);
                return nullptr;
            }
            words.insert(words.end(), {q_offsets[i], (uint32_t)lq, k_offsets[i], (uint32_t)lk});
            for (uint32_t b = 0; b < (lq * share + 31) / 32; b++) items.push_back({i, b});
        }
        // Long sequences first: a short one then ends the call.
        std::stable_sort(items.begin(), items.end(), [&](const Item &x, const Item &y) {
            return words[4 * x.sequence + 3] > words[4 * y.sequence + 3];
        });
        // A launch holds fewer than 2^32 threads.
        if (items.size() * kv_heads >= (1u << 24)) {
            h3_set_error(g, "sequences: more rows than a launch takes");
            return nullptr;
        }
        for (const Item &x : items) words.insert(words.end(), {x.sequence, x.block});
        s = new h3_hip_sequences{g, heads, kv_heads, count, (uint32_t)items.size(), q_offsets[count], k_offsets[count], nullptr};
    } catch (const std::bad_alloc &) {
        h3_set_error(g, "sequences: out of host memory");
        return nullptr;
    }
    s->table = h3_gpu_tensor_from_u32(g, words.data(), words.size());
    if (!s->table) {
        delete s;
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
    if (!s->items) return 1;
    const SeqArgs a{(uint16_t *)out->data, (const uint16_t *)q->data, (const uint16_t *)k->data, (const uint16_t *)v->data,
                    (const Sequence *)s->table->data, (const Item *)((const uint32_t *)s->table->data + 4 * (size_t)s->count),
                    s->items, s->heads, s->kv_heads, s->heads / s->kv_heads, bf16_to_f32(f32_to_bf16(scale)) * 1.4426950408889634f,
                    g->fault};
    if (!launch(g, a)) return 0;
    g->stats.attention_dispatches++;
    return 1;
}
