// Block-scaled FP8 projections (fp8_block.h): y[M,N] = bf16(sum_b 2^(ex[m,b] + ew[n/128,b])
// sum_{k in b} x8[m,k] w8[n,k] + bias), FP32 sums.
//
// The scales go into v_mfma_scale_f32_32x32x64_f8f6f4 with the codes: a lane's scale
// registers hold the bytes of its row of W and of X, the same for all K of a block, so the
// products cost what unscaled ones do. The matrix core adds the 64 products of an instruction
// with about 14 bits behind the largest (1.5e-5 of the result's root mean square, measured for
// normal values; all of its FP8 instructions do); across instructions sums are FP32.
#include "fp8_block.h"
#include "internal.h"
#include <algorithm>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr unsigned TK = FP8_BLOCK;            // K bytes of a step: one block of scales

__device__ inline unsigned swz(unsigned row, unsigned ch) { return ch ^ ((row >> 1) & 7); }

__device__ inline __amdgpu_buffer_rsrc_t uniform_resource(const void *p, unsigned bytes) {
    const uint64_t v = (uint64_t)p;
    // readfirstlane returns int: through uint32_t, so that the low word's sign stays out of the high one.
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void *)(lo | (uint64_t)hi << 32), (short)0,
                                             (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// Four columns of an output row.
__device__ inline void store4(const Fp8BlockGemmArgs &a, unsigned row, unsigned col, f32x4 v) {
    if (row >= a.m || col >= a.n) return;
    const size_t at = (size_t)row * a.n + col;
    const bool whole = a.n % 4 == 0;
    if (a.y32) {
        if (whole) *reinterpret_cast<f32x4 *>(a.y32 + at) = v;
        else
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (col + e < a.n) a.y32[at + e] = v[e];
        return;
    }
    if (a.bias)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += bf16_to_f32(a.bias[min(col + e, a.n - 1)]);
    u16x4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(v[e]);
    if (whole) *reinterpret_cast<u16x4 *>(a.y + at) = o;
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (col + e < a.n) a.y[at + e] = o[e];
}

// Row of W that row r of a tile holds, counted from the tile's first row. SwiGLU: 32 gate
// rows and the 32 up rows of the same columns alternate, so that a lane's accumulator blocks
// hold both; a tile then makes 128 columns, one block of the packed result.
__device__ inline unsigned swiglu_row(unsigned r) { return r / 64 * 32 + r % 32; }

template <int WAVES> struct RowMax { unsigned value[WAVES][64]; };

// ---------------------------------------------------------------- tiles of 128 rows
// Eight waves of 64 x 64 outputs (C^T = W . X^T), operands from memory to LDS without
// registers, three stages of 128 bytes of K. The scales of 32 steps come to LDS together.
constexpr int MID_M = 128, MID_N = 256, MID_T = 512, MID_STAGES = 3;
constexpr unsigned MID_X = MID_M * TK, MID_W = MID_N * TK, MID_STAGE = MID_X + MID_W;
constexpr unsigned SCALE_STEPS = 32;          // steps whose scales are loaded together
constexpr unsigned MID_SCALES = MID_M * SCALE_STEPS + 1024, MID_LDS = MID_STAGES * MID_STAGE + 2 * MID_SCALES;
constexpr int MID_GROUP = 4;

template <int N> __device__ inline void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The epilogue of a wave's 64 x 64 sums: row block j (32 rows), column blocks 0 and 1.
// SwiGLU: the four waves of a row meet in `most` for the block's largest magnitude.
__device__ inline void mid_epilogue(const Fp8BlockGemmArgs &a, unsigned m0, unsigned n0, unsigned wm, unsigned wn,
                                    unsigned lane, unsigned j, f32x16 c0, f32x16 c1, unsigned (*most)[4][32]) {
    const unsigned n32 = lane % 32, hf = lane / 32, row = m0 + wm * 64 + j * 32 + n32;
    if (!a.swiglu) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            store4(a, row, n0 + wn * 64 + g * 8 + hf * 4, f32x4{c0[4 * g], c0[4 * g + 1], c0[4 * g + 2], c0[4 * g + 3]});
            store4(a, row, n0 + wn * 64 + 32 + g * 8 + hf * 4, f32x4{c1[4 * g], c1[4 * g + 1], c1[4 * g + 2], c1[4 * g + 3]});
        }
        return;
    }
    float v[16];
    unsigned amax = 0;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        v[e] = swiglu_exact(c0[e], c1[e]);
        amax = max(amax, finite_magnitude(v[e], bad));
    }
    if (bad && row < a.m) *a.out.fault = 1u;
    amax = max(amax, (unsigned)__shfl_xor((int)amax, 32, 64));
    if (hf == 0) most[wm][wn][n32] = amax;
    __syncthreads();
    const unsigned scale = fp8_block_scale(max(max(most[wm][0][n32], most[wm][1][n32]), max(most[wm][2][n32], most[wm][3][n32])));
    __syncthreads();
    if (row >= a.m) return;
    const float inverse = fp8_block_inverse(scale);
    uint8_t *dst = a.out.codes + (size_t)row * a.out.stride + n0 / 2 + wn * 32 + hf * 4;
#pragma unroll
    for (int g = 0; g < 4; g++) *reinterpret_cast<unsigned *>(dst + g * 8) = fp8_block_encode4(v + 4 * g, inverse);
    if (wn == 0 && hf == 0) a.out.scales[(size_t)row * a.out.scale_stride + n0 / 256] = (uint8_t)scale;
}

__global__ __attribute__((amdgpu_flat_work_group_size(MID_T, MID_T), amdgpu_waves_per_eu(2, 2)))
void fp8_block_mid(Fp8BlockGemmArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ unsigned most[2][4][32];
    const unsigned tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const unsigned n32 = lane % 32, hf = lane / 32, wm = wave / 4, wn = wave % 4;
    unsigned ksteps = a.k / TK;
    const TileShare t = tile_share(a.tile, ksteps);
    ksteps = __builtin_amdgcn_readfirstlane(ksteps);
    const unsigned first = __builtin_amdgcn_readfirstlane(t.first), k0 = first * TK;
    unsigned tm, tn;
    band_tile((a.m + MID_M - 1) / MID_M, (a.n + MID_N - 1) / MID_N, MID_GROUP, t.pid, tm, tn);
    const unsigned m0 = __builtin_amdgcn_readfirstlane(tm * MID_M), n0 = __builtin_amdgcn_readfirstlane(tn * MID_N);

    // Rows past M or N are past the resources' size and load zeros. SwiGLU: a wave loads
    // eight rows at a time, all gate or all up rows.
    const unsigned half = a.swiglu && wave / 4 % 2, w_first = a.swiglu ? n0 / 2 + (half ? a.n / 2 : 0) : n0;
    const unsigned xrows = min(a.m - m0, (unsigned)MID_M), wrows = a.swiglu ? 128u : min(a.n - n0, (unsigned)MID_N);
    const __amdgpu_buffer_rsrc_t xr = uniform_resource(a.x + (size_t)m0 * a.k + k0, xrows * a.k - k0);
    const __amdgpu_buffer_rsrc_t wr = uniform_resource(a.w + (size_t)w_first * a.k + k0, wrows * a.k - k0);
    const unsigned lrow = 8 * wave + lane / 8, part = swz(lrow, lane % 8) * 16;
    unsigned xoff[2], woff[4];
#pragma unroll
    for (int b = 0; b < 2; b++) xoff[b] = (lrow + 64 * b) * a.k + part;
#pragma unroll
    for (int b = 0; b < 4; b++) woff[b] = (a.swiglu ? swiglu_row(lrow + 64 * b) : lrow + 64 * b) * a.k + part;
    // Scales: 16-byte parts of 32 steps from the aligned one below the first; waves 0 to 3 the
    // rows of X, wave 4 the two blocks of W in lanes 0 to 3.
    const unsigned skip = first % 16, sbase = first - skip;
    const unsigned xs_bytes = xrows * a.scale_stride - sbase;
    const __amdgpu_buffer_rsrc_t xsr = uniform_resource(a.xs + (size_t)m0 * a.scale_stride + sbase, xs_bytes);
    const unsigned wblocks = (a.n + 127) / 128;
    const __amdgpu_buffer_rsrc_t wsr = uniform_resource(a.ws + sbase, wblocks * a.scale_stride - sbase);
    const unsigned sb0 = a.swiglu ? n0 / 256 : n0 / 128, sb1 = a.swiglu ? n0 / 256 + a.n / 256 : min(n0 / 128 + 1, wblocks - 1);
    const unsigned soff = wave < 4 ? (wave * 32 + lane / 2) * a.scale_stride + lane % 2 * 16
                          : lane < 4 ? (lane / 2 ? sb1 : sb0) * a.scale_stride + lane % 2 * 16 : BUFFER_OOB;
    uint8_t *const scs = lds + MID_STAGES * MID_STAGE;
    auto load_scales = [&](unsigned group) {
        if (wave > 4) return;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            wave < 4 ? xsr : wsr, (__attribute__((address_space(3))) void *)(scs + (group & 1) * MID_SCALES + wave * 1024),
            16, soff == BUFFER_OOB ? soff : soff + group * SCALE_STEPS, 0, 0, 0);
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = f32x16{};

    // Loads of step kt into stage st; steps past the end reload the last one into a stage
    // that nobody reads again.
    auto load = [&](unsigned kt, unsigned st) {
        kt = __builtin_amdgcn_readfirstlane(min(kt, ksteps - 1));
        uint8_t *dst = lds + st * MID_STAGE + wave * 1024;
#pragma unroll
        for (int b = 0; b < 2; b++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (__attribute__((address_space(3))) void *)(dst + b * 8192), 16,
                                                     xoff[b], kt * TK, 0, 0);
#pragma unroll
        for (int b = 0; b < 4; b++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void *)(dst + MID_X + b * 8192),
                                                     16, woff[b], kt * TK, 0, 0);
    };
    auto fragment = [&](const uint8_t *tile, unsigned r, int ks) {
        const u32x4 lo = *reinterpret_cast<const u32x4 *>(tile + r * TK + swz(r, 4 * ks + 2 * hf) * 16);
        const u32x4 hi = *reinterpret_cast<const u32x4 *>(tile + r * TK + swz(r, 4 * ks + 2 * hf + 1) * 16);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    auto frags = [&](unsigned st, int ks, i32x8 *wf, i32x8 *xf) {
        const uint8_t *xs = lds + st * MID_STAGE, *ws = xs + MID_X;
#pragma unroll
        for (int i = 0; i < 2; i++) wf[i] = fragment(ws, wn * 64 + i * 32 + n32, ks);
#pragma unroll
        for (int j = 0; j < 2; j++) xf[j] = fragment(xs, wm * 64 + j * 32 + n32, ks);
    };
    int ws[2], xs[2];
    auto scales = [&](unsigned kt) {
        const unsigned at = kt + skip;
        const uint8_t *s = scs + at / SCALE_STEPS % 2 * MID_SCALES + at % SCALE_STEPS;
#pragma unroll
        for (int j = 0; j < 2; j++) xs[j] = s[(wm * 64 + j * 32 + n32) * SCALE_STEPS];
#pragma unroll
        for (int i = 0; i < 2; i++) ws[i] = s[4096 + (a.swiglu ? i : wn / 2) * SCALE_STEPS];
    };

    load_scales(0);
    load_scales(1);
#pragma unroll
    for (int s = 0; s < MID_STAGES - 1; s++) load(s, s);
    step_barrier<0>();
    i32x8 wf[2][2], xf[2][2];
    frags(0, 0, wf[0], xf[0]);
    scales(0);
    unsigned cur = 0;
    for (unsigned kt = 0; kt < ksteps; kt++) {
        const unsigned next = cur + 1 == MID_STAGES ? 0 : cur + 1, last = cur == 0 ? MID_STAGES - 1 : cur - 1;
        if (kt && (kt + skip) % SCALE_STEPS == 0) load_scales((kt + skip) / SCALE_STEPS + 1);
        load(kt + MID_STAGES - 1, last);
        frags(cur, 1, wf[1], xf[1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[0][i], xf[0][j], acc[i][j], 0, 0, 0, ws[i], 0, xs[j]);
        step_barrier<(MID_STAGES - 2) * 6>();
        frags(next, 0, wf[0], xf[0]);
        const int ws1[2] = {ws[0], ws[1]}, xs1[2] = {xs[0], xs[1]};
        scales(kt + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[1][i], xf[1][j], acc[i][j], 0, 0, 0, ws1[i], 0, xs1[j]);
        cur = next;
    }
    wait_vm_loads();   // LDS must not be written after the workgroup has ended

    if (t.partial) {
        f32x4 *dst = reinterpret_cast<f32x4 *>(a.tile.part) +
                     ((size_t)t.tile * a.tile.split + t.share) * (MID_M * MID_N / 4) + tid;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (m0 + wm * 64 + j * 32 >= a.m) break;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    dst[((j * 2 + i) * 4 + g) * MID_T] = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                                                               acc[i][j][4 * g + 3]};
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 2; j++) mid_epilogue(a, m0, n0, wm, wn, lane, j, acc[0][j], acc[1][j], most);
}

// The split tiles' shares added in order, and the epilogue. One workgroup per (tile, row block).
__global__ __launch_bounds__(MID_T) void fp8_block_mid_reduce(Fp8BlockGemmArgs a) {
    __shared__ unsigned most[2][4][32];
    const unsigned tile = blockIdx.x / 2, j = blockIdx.x % 2, tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    unsigned tm, tn;
    band_tile((a.m + MID_M - 1) / MID_M, (a.n + MID_N - 1) / MID_N, MID_GROUP, split_tile(a.tile, tile), tm, tn);
    const f32x4 *src = reinterpret_cast<const f32x4 *>(a.tile.part) + (size_t)tile * a.tile.split * (MID_M * MID_N / 4) +
                       j * 8 * MID_T + tid;
    const bool rows = tm * MID_M + wave / 4 * 64 + j * 32 < a.m;   // else no share was written
    f32x16 c[2] = {};
    for (unsigned s = 0; rows && s < a.tile.split; s++, src += MID_M * MID_N / 4)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const f32x4 v = src[(i * 4 + g) * MID_T];
#pragma unroll
                for (int e = 0; e < 4; e++) c[i][4 * g + e] += v[e];
            }
    mid_epilogue(a, tm * MID_M, tn * MID_N, wave / 4, wave % 4, lane, j, c[0], c[1], most);
}

int launch_mid(h3_gpu *g, Fp8BlockGemmArgs a, unsigned split) {
    static bool configured = false;
    if (!configured) {
        if (!h3_hip_check(g, hipFuncSetAttribute((const void *)fp8_block_mid, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 MID_LDS), "FP8 block GEMM shared memory"))
            return 0;
        configured = true;
    }
    const unsigned tiles = (a.m + MID_M - 1) / MID_M * ((a.n + MID_N - 1) / MID_N);
    a.tile = split_last_wave(g, tiles, split, a.k / TK, MID_M * MID_N);
    const unsigned rest = tiles - a.tile.full;
    h3_note_kernel(g, "fp8_block_mid", MID_M, a.tile.split);
    hipEvent_t timing = h3_kernel_timing_begin(g);
    hipLaunchKernelGGL(fp8_block_mid, dim3(a.tile.full + rest * a.tile.split), dim3(MID_T), MID_LDS, g->compute, a);
    if (rest && h3_launch_status(g, "FP8 block GEMM"))
        hipLaunchKernelGGL(fp8_block_mid_reduce, dim3(rest * 2), dim3(MID_T), 0, g->compute, a);
    h3_kernel_timing_end(g, timing);
    return h3_launch_status(g, "FP8 block GEMM");
}

}  // namespace

bool h3_gemm_fp8_block_fuses(const h3_gpu *g, uint32_t m) { return m > 0 && g; }

int h3_gemm_fp8_block(h3_gpu *g, const Fp8BlockGemmArgs &a) {
    return launch_mid(g, a, 1);
}
