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
#include <type_traits>

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr unsigned TK = FP8_BLOCK;            // K bytes of a step: one block of scales

__device__ inline unsigned swz(unsigned row, unsigned ch) { return ch ^ ((row >> 1) & 7); }

// A buffer resource in scalar registers. Raw: loads past `bytes` give zeros.
__device__ inline i32x4 asm_resource(const uint8_t *p, unsigned bytes) {
    const uint64_t v = (uint64_t)p;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((unsigned)v), (int)__builtin_amdgcn_readfirstlane((unsigned)(v >> 32)),
                 (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}

// Epilogues: BF16 rows of a multiple of eight columns, without and with a bias; SwiGLU, packed;
// any columns, BF16 (with or without a bias); and the FP32 sums (few rows only). Kernels are
// instantiated for each: the epilogue is straight-line code that runs once per tile, and one that
// branches between them is 100 KB of it for 256 x 256 tiles (18225 rows, 5376 -> 28672: 1.3% slower).
enum { EPI_PLAIN = 0, EPI_BIAS = 1, EPI_SWIGLU = 2, EPI_ANY = 3, EPI_SUMS = 4 };
int epilogue_of(const Fp8BlockGemmArgs &a) {
    return a.swiglu ? EPI_SWIGLU : a.y32 ? EPI_SUMS : a.n % 8 ? EPI_ANY : a.bias ? EPI_BIAS : EPI_PLAIN;
}

// Four values wherever they lie: global loads and stores need no alignment.
struct __attribute__((packed, aligned(2))) u16x4_any { uint16_t v[4]; };
struct __attribute__((packed, aligned(2))) u16x2_any { uint16_t v[2]; };
struct __attribute__((packed, aligned(2))) u32x4_any { u32x4 v; };

// Four columns of an output row.
template <int EPI>
__device__ inline void store4(const Fp8BlockGemmArgs &a, unsigned row, unsigned col, f32x4 v) {
    if (row >= a.m || col >= a.n) return;
    const size_t at = (size_t)row * a.n + col;
    if constexpr (EPI == EPI_SUMS) {       // the MLP's: a multiple of four columns
        *reinterpret_cast<f32x4 *>(a.y32 + at) = v;
        return;
    }
    if constexpr (EPI == EPI_ANY) {
        const bool whole = col + 4 <= a.n;
        u16x4_any b = {};
        if (a.bias) {
            if (whole) b = *reinterpret_cast<const u16x4_any *>(a.bias + col);
            else
#pragma unroll
                for (unsigned e = 0; e < 3; e++) b.v[e] = a.bias[min(col + e, a.n - 1)];
        }
        u16x4_any o;
#pragma unroll
        for (int e = 0; e < 4; e++) o.v[e] = f32_to_bf16(v[e] + bf16_to_f32(b.v[e]));
        if (whole) *reinterpret_cast<u16x4_any *>(a.y + at) = o;
        else
#pragma unroll
            for (unsigned e = 0; e < 3; e++)
                if (col + e < a.n) a.y[at + e] = o.v[e];
        return;
    }
    if constexpr (EPI == EPI_BIAS) {
        const u16x4 b = *reinterpret_cast<const u16x4 *>(a.bias + col);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += bf16_to_f32(b[e]);
    }
    u16x4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(v[e]);
    *reinterpret_cast<u16x4 *>(a.y + at) = o;
}

// ---------------------------------------------------------------- few rows
// Reading W once is all the work there is, so the split is made for memory: a workgroup takes
// 16 NB columns of 16 RB rows (rows: one workgroup's wherever W is large), and its waves take
// the K steps in turn, so that together they read consecutive bytes of every weight row,
// straight into registers; their sums meet in LDS, added in wave order. x and the scales come
// from L2, which all workgroups share, as the operands of v_mfma_scale_f32_16x16x128_f8f6f4.
// PACK: x is BF16 and every workgroup packs it for itself, where that is less than the launch it
// saves (1 row, 256 -> 5376: 4.3 us, 8.0 with a launch of its own).
//
// HBM-bound: 1 row, 5376 -> 32256 (173 MB): 32 us, 5.4 TB/s, 4 us of them a launch's; 16 rows
// 36, as x's reads weigh more. One row of the tile kernels: 37.
template <int RB, int NB, int WAVES> constexpr int stream_lds() { return WAVES * NB * RB * 64 * 16; }

template <int EPI, bool PACK, int RB, int NB, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void fp8_block_stream(Fp8BlockGemmArgs a, unsigned groups) {
    static_assert(U == 2 || U == 3, "steps of a call");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const unsigned tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
    const unsigned r = lane % 16, q = lane / 16, pid = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned n0 = pid / groups * 16 * NB, m0 = pid % groups * 16 * RB, steps = a.k / TK;
    // Rows past M and columns past N repeat the last one; not stored. An operand's 32 bytes of a
    // step are two 16-byte pieces that lie beside those of the row's other lanes (which K value
    // of the step a byte is does not matter where W and x agree).
    using X = std::conditional_t<PACK, uint16_t, uint8_t>;
    constexpr int XV = 2 * sizeof(X);         // 16-byte loads of an operand of x
    const X *xp[RB];
    const uint8_t *wp[NB], *xsp[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) {
        const unsigned row = min(m0 + i * 16 + r, a.m - 1);
        if constexpr (PACK) {
            xp[i] = a.xb + (size_t)row * a.columns + 16 * q;
        } else {
            xp[i] = a.x + (size_t)row * a.k + 16 * q;
            xsp[i] = a.xs + fp8_block_scale_at(row, 0, a.groups);
        }
    }
#pragma unroll
    for (int i = 0; i < NB; i++) wp[i] = a.w + (size_t)min(n0 + i * 16 + r, a.n - 1) * a.k + 16 * q;
    const uint8_t *wsp = a.ws + fp8_block_scale_at(n0 / FP8_BLOCK, 0, a.groups);
    f32x4 acc[NB][RB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < RB; j++) acc[i][j] = f32x4{};

    // BF16 values of a step, as fp8_block_pack packs them: a row's four lanes hold a block. (A
    // last block that is cut off is loaded whole: up to 254 bytes behind the last row, which a
    // tensor's allocation has.)
    auto pack = [&](unsigned step, u32x4 *x) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; e++) {
            const unsigned word = x[e / 8][e % 8 / 2];
            v[e] = __builtin_bit_cast(float, e % 2 ? word & 0xffff0000u : word << 16);
        }
        if ((step + 1) * TK > a.columns)      // the last block is cut off
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (step * TK + 64 * (e / 16) + 16 * q + e % 16 >= a.columns) v[e] = 0.f;
        bool bad = false;
        unsigned amax = fp8_block_magnitude<32>(v, bad);
        if (bad) *a.fault = 1u;
        amax = max(amax, (unsigned)__shfl_xor((int)amax, 16, 64));
        amax = max(amax, (unsigned)__shfl_xor((int)amax, 32, 64));
        const unsigned scale = fp8_block_scale(amax);
        const float value = fp8_block_value(scale);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int w = 0; w < 4; w++) x[h][w] = fp8_block_encode4(v + 16 * h + 4 * w, value);
        return (int)scale;
    };
    auto run = [&](unsigned s, auto count) {
        constexpr int C = decltype(count)::value;
        u32x4 w[C][NB][2], x[C][RB][XV];
        int ws[C], xs[C][RB];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const unsigned step = s + c * WAVES, at = step / 4 * 128 + step % 4;
            const size_t k = (size_t)step * TK;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) w[c][i][h] = *reinterpret_cast<const u32x4 *>(wp[i] + k + 64 * h);
            ws[c] = wsp[at];
#pragma unroll
            for (int j = 0; j < RB; j++) {
                if constexpr (!PACK) xs[c][j] = xsp[j][at];
#pragma unroll
                for (int h = 0; h < XV; h++)
                    x[c][j][h] = reinterpret_cast<const u32x4_any *>(xp[j] + k + 64 * (h * 2 / XV) + 8 * (h % (XV / 2)))->v;
            }
        }
        auto whole = [](const u32x4 *v) {
            return i32x8{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3], (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
        };
#pragma unroll
        for (int c = 0; c < C; c++) {
            if constexpr (PACK)
#pragma unroll
                for (int j = 0; j < RB; j++) xs[c][j] = pack(s + c * WAVES, x[c][j]);
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < RB; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(whole(w[c][i]), whole(x[c][j]), acc[i][j], 0, 0,
                                                                                 0, ws[c], 0, xs[c][j]);
        }
    };
    unsigned s = wave;
    for (; s + (U - 1) * WAVES < steps; s += U * WAVES) run(s, std::integral_constant<int, U>{});
    // The rest in one go too: the loads of a call are in flight together.
    const unsigned rest = s < steps ? (steps - s + WAVES - 1) / WAVES : 0;
    if constexpr (U > 2)
        if (rest == 2) run(s, std::integral_constant<int, 2>{});
    if (rest == 1) run(s, std::integral_constant<int, 1>{});

    // [wave][block][lane] of four sums.
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);
    constexpr unsigned ITEMS = NB * RB * 64;
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < RB; j++) part[wave * ITEMS + (i * RB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (unsigned at = 0; at < ITEMS; at += 64 * WAVES) {
        const unsigned item = at + tid;
        if (ITEMS % (64 * WAVES) && item >= ITEMS) break;
        f32x4 v = part[item];
#pragma unroll
        for (int w = 1; w < WAVES; w++) v += part[w * ITEMS + item];
        store4<EPI>(a, m0 + item / 64 % RB * 16 + item % 16, n0 + item / 64 / RB * 16 + item % 64 / 16 * 4, v);
    }
}

uint64_t stream_groups(const Fp8BlockGemmArgs &a, unsigned rb, unsigned nb) {
    return ((uint64_t)a.m + 16 * rb - 1) / (16 * rb) * (((uint64_t)a.n + 16 * nb - 1) / (16 * nb));
}
// Workgroups of the busiest CU.
float stream_rounds(const h3_gpu *g, const Fp8BlockGemmArgs &a, unsigned rb, unsigned nb) {
    return (float)((stream_groups(a, rb, nb) + g->cus - 1) / g->cus);
}

template <int EPI, bool PACK, int RB, int NB, int WAVES, int U>
int launch_stream_as(h3_gpu *g, const Fp8BlockGemmArgs &a) {
    constexpr int shared = stream_lds<RB, NB, WAVES>();
    static_assert(shared <= 65536, "LDS without an attribute");
    const unsigned groups = (a.m + 16 * RB - 1) / (16 * RB), columns = (a.n + 16 * NB - 1) / (16 * NB);
    h3_note_kernel(g, PACK ? "fp8_block_stream packing" : "fp8_block_stream", 16 * RB);
    hipLaunchKernelGGL((fp8_block_stream<EPI, PACK, RB, NB, WAVES, U>), dim3(columns * groups), dim3(64 * WAVES), shared,
                       g->compute, a, groups);
    return h3_launch_status(g, "FP8 block GEMM");
}
// Row blocks and column blocks of a workgroup. With 64 columns of 16 rows and more than a workgroup
// per CU, four waves of fewer registers, so that more of those run at a time (1 row, 5376 -> 32256:
// 32.2 us, eight waves 34.5; 16128 columns, a workgroup per CU: 16.5, 15.1).
template <int EPI, bool PACK> int launch_stream(h3_gpu *g, const Fp8BlockGemmArgs &a, unsigned rb, unsigned nb) {
    if (rb == 1 && nb == 2) return launch_stream_as<EPI, PACK, 1, 2, 8, 3>(g, a);
    if (rb == 1) return stream_rounds(g, a, 1, 4) > 1.f ? launch_stream_as<EPI, PACK, 1, 4, 4, 2>(g, a)
                                                        : launch_stream_as<EPI, PACK, 1, 4, 8, 2>(g, a);
    if (rb == 2) return nb == 2 ? launch_stream_as<EPI, PACK, 2, 2, 4, 3>(g, a) : launch_stream_as<EPI, PACK, 2, 4, 4, 3>(g, a);
    return launch_stream_as<EPI, PACK, 3, 2, 4, 2>(g, a);
}

// ---------------------------------------------------------------- tiles of 256 rows
// 256 x 256 outputs per workgroup, four waves of 128 x 128 (one per SIMD), each 4 x 4
// accumulator blocks of 32 x 32 in AGPRs, so that one fragment read from LDS feeds four
// MFMAs. The K loop is one inline-asm block, because its value is the order of the
// instructions; with one wave per SIMD nothing else hides a stall:
//  * a K tile is one block of 128 bytes, two substeps of sixteen MFMAs; the eight 32-byte
//    fragments of the next substep are read in the first eight MFMA slots of the current
//    one, two ds_read_b128 each, into the other register set;
//  * the sixteen global -> LDS loads of a K tile (1 KB each) are issued two tiles ahead,
//    one per MFMA of the second substep, into the stage this tile has finished reading;
//  * one barrier per tile, between the substeps;
//  * the scales of four tiles are the bytes of one dword per fragment row, loaded into the
//    other one of two register sets a group of four tiles ahead; the MFMAs of tile B of a
//    group take byte B (op_sel), so the body is two groups.
// LDS (128 KB): X stages at 0 and 32 KB, W stages at 64 and 96 KB; rows of 128 codes with
// XOR-swizzled 16-byte chunks. Fixed registers: fragment set S in v[64 + 64 S ..], W block
// I at + 8 I, X block J at + 32 + 8 J; scale set Z in v[192 + 6 Z ..], X block J at + J, W at
// + 4 (even blocks) and + 5 (odd ones: with SwiGLU those are up rows).
//
// Tiles of 128 rows are the same with waves of 64 x 128 and half as many products a tile, too
// few to cover the memory's latency with one tile of lead: three stages, X at 0, 16 and 32 KB,
// W at 48, 80 and 112 KB, and loads three tiles ahead. Fragment set S in v[64 + 48 S ..], X
// block J at + 32 + 8 J; scale set Z in v[160 + 4 Z ..], X block J at + J, W at + 2 and + 3. The
// body is 24 tiles: three stages, four bytes, two sets.
constexpr int PIPE_N = 256, PIPE_T = 256;
template <int TM> constexpr unsigned pipe_lds() { return TM == 256 ? 4 * 256 * TK : 3 * (128 + 256) * TK; }
constexpr int PIPE_GROUP = 4;
constexpr unsigned QUAD = 4;                  // K tiles whose scales are loaded together

#define FB_LX(ST, T) "s_add_u32 m0, %[mb], 32768*" #ST "+4096*" #T "\n"                                             \
    "buffer_load_dwordx4 %[x" #T "], %[sx], %[kc] offen lds\n"
#define FB_LW(ST, T, R) "s_add_u32 m0, %[mb], 65536+32768*" #ST "+4096*" #T "\n"                                    \
    "buffer_load_dwordx4 %[y" #T "], %[sw" #R "], %[kc] offen lds\n"
#define FB_LOADS(ST) FB_LX(ST, 0), FB_LW(ST, 0, 0), FB_LX(ST, 1), FB_LW(ST, 1, 1), FB_LX(ST, 2), FB_LW(ST, 2, 0),    \
    FB_LX(ST, 3), FB_LW(ST, 3, 1), FB_LX(ST, 4), FB_LW(ST, 4, 0), FB_LX(ST, 5), FB_LW(ST, 5, 1), FB_LX(ST, 6),         \
    FB_LW(ST, 6, 0), FB_LX(ST, 7), FB_LW(ST, 7, 1)
#define FB_NONE "", "", "", "", "", "", "", "", "", "", "", "", "", "", "", ""
// The scales of the group at byte kg of a run of rows into set Z.
#define FB_SCALES(Z)                                                                                                \
    "buffer_load_dword v[192+6*" #Z "], %[e0], %[tx], %[kg] offen\n"                                                 \
    "buffer_load_dword v[192+6*" #Z "+1], %[e1], %[tx], %[kg] offen\n"                                               \
    "buffer_load_dword v[192+6*" #Z "+2], %[e2], %[tx], %[kg] offen\n"                                               \
    "buffer_load_dword v[192+6*" #Z "+3], %[e3], %[tx], %[kg] offen\n"                                               \
    "buffer_load_dword v[192+6*" #Z "+4], %[e4], %[tw], %[kg] offen\n"                                               \
    "buffer_load_dword v[192+6*" #Z "+5], %[e5], %[tw], %[kg] offen\n"                                               \
    "s_add_u32 %[kg], %[kg], 128\n"                                                                                 \
    "s_min_u32 %[kg], %[kg], %[kgmax]\n"
#define FB_SEL_0 " op_sel:[0,0,0] op_sel_hi:[0,0,0]\n"
#define FB_SEL_1 " op_sel:[1,1,0] op_sel_hi:[0,0,0]\n"
#define FB_SEL_2 " op_sel:[0,0,0] op_sel_hi:[1,1,0]\n"
#define FB_SEL_3 " op_sel:[1,1,0] op_sel_hi:[1,1,0]\n"
#define FB_MFMA(S, Z, B, I, J, P)                                                                                   \
    "v_mfma_scale_f32_32x32x64_f8f6f4 %[c" #I #J "], v[64+64*" #S "+8*" #I ":64+64*" #S "+8*" #I "+7], "             \
    "v[64+64*" #S "+32+8*" #J ":64+64*" #S "+32+8*" #J "+7], %[c" #I #J "], v[192+6*" #Z "+4+" #P "], "              \
    "v[192+6*" #Z "+" #J "]" FB_SEL_##B
// Fragment F of substep KS, stage ST, into set T: its two 16-byte halves.
#define FB_RW(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+64*" #T "+8*" #F ":64+64*" #T "+8*" #F "+3], %[w" #KS "0] offset:32768*" #ST "+4096*" #F "\n"     \
    "ds_read_b128 v[64+64*" #T "+8*" #F "+4:64+64*" #T "+8*" #F "+7], %[w" #KS "1] offset:32768*" #ST "+4096*" #F "\n"
#define FB_RX(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+64*" #T "+32+8*" #F ":64+64*" #T "+32+8*" #F "+3], %[r" #KS "0] offset:32768*" #ST "+4096*" #F "\n" \
    "ds_read_b128 v[64+64*" #T "+32+8*" #F "+4:64+64*" #T "+32+8*" #F "+7], %[r" #KS "1] offset:32768*" #ST "+4096*" #F "\n"
// A substep of set S with scale set Z, byte B, that reads substep KS of stage ST into set T;
// L0..L15 behind its MFMAs.
#define FB_SUB(S, Z, B, T, KS, ST, L0, L1, L2, L3, L4, L5, L6, L7, L8, L9, L10, L11, L12, L13, L14, L15)              \
    FB_MFMA(S, Z, B, 0, 0, 0) FB_RW(T, 0, KS, ST) L0 FB_MFMA(S, Z, B, 0, 1, 0) FB_RX(T, 0, KS, ST) L1                \
    FB_MFMA(S, Z, B, 0, 2, 0) FB_RX(T, 1, KS, ST) L2 FB_MFMA(S, Z, B, 0, 3, 0) FB_RX(T, 2, KS, ST) L3                \
    FB_MFMA(S, Z, B, 1, 0, 1) FB_RX(T, 3, KS, ST) L4 FB_MFMA(S, Z, B, 1, 1, 1) FB_RW(T, 1, KS, ST) L5                \
    FB_MFMA(S, Z, B, 1, 2, 1) FB_RW(T, 2, KS, ST) L6 FB_MFMA(S, Z, B, 1, 3, 1) FB_RW(T, 3, KS, ST) L7                \
    FB_MFMA(S, Z, B, 2, 0, 0) L8 FB_MFMA(S, Z, B, 2, 1, 0) L9 FB_MFMA(S, Z, B, 2, 2, 0) L10                          \
    FB_MFMA(S, Z, B, 2, 3, 0) L11 FB_MFMA(S, Z, B, 3, 0, 1) L12 FB_MFMA(S, Z, B, 3, 1, 1) L13                        \
    FB_MFMA(S, Z, B, 3, 2, 1) L14 FB_MFMA(S, Z, B, 3, 3, 1) L15
#define FB_SUB_EXP(...) FB_SUB(__VA_ARGS__)
// K tile B of a group in stage ST, next tile's stage OT; NEXT: loads of the next group's scales.
#define FB_TILE(ST, OT, Z, B, NEXT)                                                                                 \
    FB_SUB_EXP(0, Z, B, 1, 1, ST, FB_NONE)                                                                           \
    "s_waitcnt vmcnt(0) lgkmcnt(0)\n"                                                                               \
    "s_barrier\n"                                                                                                   \
    "s_min_u32 %[kc], %[kn], %[kmax]\n"                                                                             \
    "s_add_u32 %[kn], %[kn], 128\n" NEXT                                                                            \
    FB_SUB_EXP(1, Z, B, 0, 0, OT, FB_LOADS(ST))                                                                      \
    "s_waitcnt lgkmcnt(0)\n"                                                                                        \
    "s_sub_u32 %[steps], %[steps], 1\n"                                                                             \
    "s_cmp_eq_u32 %[steps], 0\n"                                                                                    \
    "s_cbranch_scc1 fb_end_%=\n"
#define FB_QUAD(Z, OZ) FB_TILE(0, 1, Z, 0, FB_SCALES(OZ)) FB_TILE(1, 0, Z, 1, "") FB_TILE(0, 1, Z, 2, "") FB_TILE(1, 0, Z, 3, "")
#define FB_FIRST(ST, KC) "s_mov_b32 %[kc], " KC "\n" FB_LX(ST, 0) FB_LW(ST, 0, 0) FB_LX(ST, 1) FB_LW(ST, 1, 1)           \
    FB_LX(ST, 2) FB_LW(ST, 2, 0) FB_LX(ST, 3) FB_LW(ST, 3, 1) FB_LX(ST, 4) FB_LW(ST, 4, 0) FB_LX(ST, 5) FB_LW(ST, 5, 1) \
    FB_LX(ST, 6) FB_LW(ST, 6, 0) FB_LX(ST, 7) FB_LW(ST, 7, 1)
// Tiles of 128 rows.
#define FH_LX(ST, T) "s_add_u32 m0, %[mb], 16384*" #ST "+4096*" #T "\n"                                             \
    "buffer_load_dwordx4 %[x" #T "], %[sx], %[kc] offen lds\n"
#define FH_LW(ST, T, R) "s_add_u32 m0, %[mb], 49152+32768*" #ST "+4096*" #T "\n"                                    \
    "buffer_load_dwordx4 %[y" #T "], %[sw" #R "], %[kc] offen lds\n"
#define FH_SCALES(Z)                                                                                                \
    "buffer_load_dword v[160+4*" #Z "], %[e0], %[tx], %[kg] offen\n"                                                 \
    "buffer_load_dword v[160+4*" #Z "+1], %[e1], %[tx], %[kg] offen\n"                                               \
    "buffer_load_dword v[160+4*" #Z "+2], %[e4], %[tw], %[kg] offen\n"                                               \
    "buffer_load_dword v[160+4*" #Z "+3], %[e5], %[tw], %[kg] offen\n"                                               \
    "s_add_u32 %[kg], %[kg], 128\n"                                                                                 \
    "s_min_u32 %[kg], %[kg], %[kgmax]\n"
#define FH_MFMA(S, Z, B, I, J, P)                                                                                   \
    "v_mfma_scale_f32_32x32x64_f8f6f4 %[c" #I #J "], v[64+48*" #S "+8*" #I ":64+48*" #S "+8*" #I "+7], "             \
    "v[64+48*" #S "+32+8*" #J ":64+48*" #S "+32+8*" #J "+7], %[c" #I #J "], v[160+4*" #Z "+2+" #P "], "              \
    "v[160+4*" #Z "+" #J "]" FB_SEL_##B
// W's stage ST is within a ds_read's offset of base 0 (stages 0 and 1) or of its own (2).
#define FH_WAT_0(KS, H) "%[w" #KS #H "] offset:"
#define FH_WAT_1(KS, H) "%[w" #KS #H "] offset:32768+"
#define FH_WAT_2(KS, H) "%[u" #KS #H "] offset:"
#define FH_RW(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+48*" #T "+8*" #F ":64+48*" #T "+8*" #F "+3], " FH_WAT_##ST(KS, 0) "4096*" #F "\n"              \
    "ds_read_b128 v[64+48*" #T "+8*" #F "+4:64+48*" #T "+8*" #F "+7], " FH_WAT_##ST(KS, 1) "4096*" #F "\n"
#define FH_RX(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+48*" #T "+32+8*" #F ":64+48*" #T "+32+8*" #F "+3], %[r" #KS "0] offset:16384*" #ST "+4096*" #F "\n" \
    "ds_read_b128 v[64+48*" #T "+32+8*" #F "+4:64+48*" #T "+32+8*" #F "+7], %[r" #KS "1] offset:16384*" #ST "+4096*" #F "\n"
#define FH_SUB(S, Z, B, T, KS, ST, L0, L1, L2, L3, L4, L5, L6, L7)                                                    \
    FH_MFMA(S, Z, B, 0, 0, 0) FH_RW(T, 0, KS, ST) L0 FH_MFMA(S, Z, B, 0, 1, 0) FH_RX(T, 0, KS, ST) L1                \
    FH_MFMA(S, Z, B, 1, 0, 1) FH_RX(T, 1, KS, ST) L2 FH_MFMA(S, Z, B, 1, 1, 1) FH_RW(T, 1, KS, ST) L3                \
    FH_MFMA(S, Z, B, 2, 0, 0) FH_RW(T, 2, KS, ST) L4 FH_MFMA(S, Z, B, 2, 1, 0) FH_RW(T, 3, KS, ST) L5                \
    FH_MFMA(S, Z, B, 3, 0, 1) L6 FH_MFMA(S, Z, B, 3, 1, 1) L7
#define FH_SUB_EXP(...) FH_SUB(__VA_ARGS__)
#define FH_NONE "", "", "", "", "", "", "", ""
#define FH_LOADS(ST) FH_LX(ST, 0), FH_LW(ST, 0, 0), FH_LX(ST, 1), FH_LW(ST, 1, 1), FH_LX(ST, 2) FH_LW(ST, 2, 0),      \
    FH_LX(ST, 3) FH_LW(ST, 3, 1), FH_LW(ST, 4, 0) FH_LW(ST, 5, 1), FH_LW(ST, 6, 0) FH_LW(ST, 7, 1)
// The loads of the tile after next (12, the youngest) stay in flight at the barrier.
#define FH_TILE(ST, OT, Z, B, NEXT)                                                                                 \
    FH_SUB_EXP(0, Z, B, 1, 1, ST, FH_NONE)                                                                           \
    "s_waitcnt vmcnt(12) lgkmcnt(0)\n"                                                                              \
    "s_barrier\n"                                                                                                   \
    "s_min_u32 %[kc], %[kn], %[kmax]\n"                                                                             \
    "s_add_u32 %[kn], %[kn], 128\n" NEXT                                                                            \
    FH_SUB_EXP(1, Z, B, 0, 0, OT, FH_LOADS(ST))                                                                      \
    "s_waitcnt lgkmcnt(0)\n"                                                                                        \
    "s_sub_u32 %[steps], %[steps], 1\n"                                                                             \
    "s_cmp_eq_u32 %[steps], 0\n"                                                                                    \
    "s_cbranch_scc1 fh_end_%=\n"
// Four tiles from stage S0 on.
#define FH_QUAD(S0, S1, S2, Z, OZ) FH_TILE(S0, S1, Z, 0, FH_SCALES(OZ)) FH_TILE(S1, S2, Z, 1, "")                     \
    FH_TILE(S2, S0, Z, 2, "") FH_TILE(S0, S1, Z, 3, "")
#define FH_FIRST(ST, KC) "s_mov_b32 %[kc], " KC "\n" FH_LX(ST, 0) FH_LW(ST, 0, 0) FH_LX(ST, 1) FH_LW(ST, 1, 1)           \
    FH_LX(ST, 2) FH_LW(ST, 2, 0) FH_LX(ST, 3) FH_LW(ST, 3, 1) FH_LW(ST, 4, 0) FH_LW(ST, 5, 1) FH_LW(ST, 6, 0) FH_LW(ST, 7, 1)
#define FH_ACC2(I) [c##I##0] "+a"(c[I][0]), [c##I##1] "+a"(c[I][1])
#define FB_ACC4(I) [c##I##0] "+a"(c[I][0]), [c##I##1] "+a"(c[I][1]), [c##I##2] "+a"(c[I][2]), [c##I##3] "+a"(c[I][3])
#define FB_CL10(x) "v" #x "0", "v" #x "1", "v" #x "2", "v" #x "3", "v" #x "4", "v" #x "5", "v" #x "6", "v" #x "7",     \
    "v" #x "8", "v" #x "9"

template <int TM>
__device__ inline void pipe_tile(const Fp8BlockGemmArgs &a, unsigned pid, unsigned &m0, unsigned &n0) {
    unsigned tm, tn;
    band_tile((a.m + TM - 1) / TM, (a.n + PIPE_N - 1) / PIPE_N, PIPE_GROUP, pid, tm, tn);
    m0 = __builtin_amdgcn_readfirstlane(tm * TM);
    n0 = __builtin_amdgcn_readfirstlane(tn * PIPE_N);
}

// The workgroup's share of the K tiles: whole groups of four, so that the scales' dwords stay
// aligned. On return t.first counts tiles and ksteps is their number.
__device__ inline TileShare pipe_share(const Fp8BlockGemmArgs &a, unsigned &ksteps) {
    unsigned quads = (ksteps + QUAD - 1) / QUAD;
    TileShare t = tile_share(a.tile, quads);
    t.first *= QUAD;
    ksteps = min(quads * QUAD, ksteps - t.first);
    return t;
}

// Between a wave's writes to LDS and its own lanes' reads of them, and before it writes there
// again: no barrier, but their order stays.
__device__ inline void wave_stores_first() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 32 columns of an output row, from col, as BF16, registers as the MFMA leaves them: group g of
// lane half hf holds columns 8 g + 4 hf + 0..3. v_permlane32_swap gives the low half both halves
// of group g, the high half those of group g + 1: 16 bytes a lane.
template <int EPI>
__device__ inline void round_row(const Fp8BlockGemmArgs &a, unsigned col, unsigned hf, const f32x16 &c, uint8_t *to) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        unsigned w[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4 v = {c[4 * (g + h)], c[4 * (g + h) + 1], c[4 * (g + h) + 2], c[4 * (g + h) + 3]};
            if constexpr (EPI == EPI_BIAS) {
                const u16x4 b = *reinterpret_cast<const u16x4 *>(a.bias + min(col + 8 * (g + h) + 4 * hf, a.n - 4));
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += bf16_to_f32(b[e]);
            }
            u16x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = f32_to_bf16(v[e]);
            w[h][0] = o[0] | ((unsigned)o[1] << 16);
            w[h][1] = o[2] | ((unsigned)o[3] << 16);
        }
        const auto s0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        *reinterpret_cast<u32x4 *>(to + 16 * (g + hf)) = u32x4{s0[0], s1[0], s0[1], s1[1]};
    }
}

// 32 rows x 32 NB columns of a wave, n a multiple of 8, through LDS into whole cache lines.
//
// PAST: past the L2's resident lines. All workgroups of a wave of 256-row tiles store at once, 33
// MB; stored from the registers, 32 bytes of 32 rows an instruction, that takes 12 of a tile's 75
// us (18225 rows, 5376 -> 28672: 2385 us, 1975 without any stores); so 2132. (The lines alone:
// 2370; past the L2 alone: 2440. One card; others, or runs of other lengths, 1967 to 2184.)
template <int NB> constexpr unsigned ROW_LDS = NB * 64 + 16;    // bytes of a row in LDS, padded against bank conflicts
template <int EPI, bool PAST, int NB>
__device__ inline void store_rows(const Fp8BlockGemmArgs &a, unsigned row0, unsigned col, unsigned lane,
                                  const f32x16 *const (&c)[NB], uint8_t *rows) {
    constexpr unsigned LANES = NB * 4, STEP = 64 / LANES;       // lanes of a row, rows of an instruction
    const unsigned hf = lane / 32, row = row0 + lane / LANES, at = col + lane % LANES * 8;
    uint8_t *to = rows + lane % 32 * ROW_LDS<NB>;
#pragma unroll
    for (int i = 0; i < NB; i++) round_row<EPI>(a, col + 32 * i, hf, *c[i], to + 64 * i);
    wave_stores_first();
    const uint8_t *from = rows + lane / LANES * ROW_LDS<NB> + lane % LANES * 16;
    uint16_t *dst = a.y + (size_t)row * a.n + at;
#pragma unroll
    for (unsigned r = 0; r < 32; r += STEP) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(from + r * ROW_LDS<NB>);
        if (row + r >= a.m || at >= a.n) continue;
        u32x4 *line = reinterpret_cast<u32x4 *>(dst + (size_t)r * a.n);
        if constexpr (PAST) __builtin_nontemporal_store(v, line);
        else *line = v;
    }
    wave_stores_first();
}

// 32 rows x 128 columns of a wave through LDS, so that rows of any alignment go out whole: two
// columns a lane.
constexpr unsigned ANY_ROW = 132;             // FP32 values of a row in LDS, padded against bank conflicts
constexpr unsigned ANY_LDS = 4 * 32 * ANY_ROW * 4;
__device__ inline void pipe_any(const Fp8BlockGemmArgs &a, unsigned row0, unsigned col, unsigned lane, const f32x16 &c0,
                                const f32x16 &c1, const f32x16 &c2, const f32x16 &c3, float *rows) {
    const unsigned n32 = lane % 32, hf = lane / 32;
    const f32x16 *c[4] = {&c0, &c1, &c2, &c3};
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<f32x4 *>(rows + n32 * ANY_ROW + 32 * i + 8 * g + 4 * hf) =
                f32x4{(*c[i])[4 * g], (*c[i])[4 * g + 1], (*c[i])[4 * g + 2], (*c[i])[4 * g + 3]};
    wave_stores_first();
    const unsigned at = col + 2 * lane;
    float bias[2] = {};
    if (a.bias)
        for (unsigned e = 0; e < 2; e++) bias[e] = at + e < a.n ? bf16_to_f32(a.bias[at + e]) : 0.f;
    const unsigned count = at < a.n ? min(a.m > row0 ? a.m - row0 : 0u, 32u) : 0u;
    for (unsigned r = 0; r < count; r++) {
        const f32x2 v = *reinterpret_cast<const f32x2 *>(rows + r * ANY_ROW + 2 * lane);
        const size_t to = (size_t)(row0 + r) * a.n + at;
        const u16x2_any o = {{f32_to_bf16(v[0] + bias[0]), f32_to_bf16(v[1] + bias[1])}};
        if (at + 1 < a.n) *reinterpret_cast<u16x2_any *>(a.y + to) = o;
        else a.y[to] = o.v[0];
    }
    wave_stores_first();
}

constexpr unsigned CODE_ROW = 128 + 16, CODE_ROWS = 512;      // a row of codes in LDS, and where they begin
// The epilogue of a wave's 32 rows from row0 x 128 columns, blocks c0 to c3. SwiGLU: the
// two waves of a row meet in scratch (LDS) for the largest magnitude of its 128 columns.
template <int EPI>
__device__ inline void pipe_epilogue(const Fp8BlockGemmArgs &a, unsigned row0, unsigned n0, unsigned wm, unsigned wn,
                                     unsigned lane, const f32x16 &c0, const f32x16 &c1, const f32x16 &c2,
                                     const f32x16 &c3, void *scratch) {
    const unsigned n32 = lane % 32, hf = lane / 32, row = row0 + n32, col = n0 + wn * 128;
    auto most = (unsigned(*)[2][32])scratch;
    if constexpr (EPI == EPI_ANY) {
        pipe_any(a, row0, col, lane, c0, c1, c2, c3, (float *)scratch + (wm * 2 + wn) * 32 * ANY_ROW);
        return;
    }
    if constexpr (EPI != EPI_SWIGLU) {
        store_rows<EPI, true, 4>(a, row0, col, lane, {&c0, &c1, &c2, &c3}, (uint8_t *)scratch + (wm * 2 + wn) * 32 * ROW_LDS<4>);
        return;
    }
    float v[32];
    bool bad = false;
    float gate[32], up[32];
#pragma unroll
    for (int e = 0; e < 16; e++) {
        gate[e] = c0[e];
        up[e] = c1[e];
        gate[16 + e] = c2[e];
        up[16 + e] = c3[e];
    }
    swiglu<32, true>(gate, up, v);
    unsigned amax = fp8_block_magnitude<32>(v, bad);
    if (bad && row < a.m) *a.out.fault = 1u;
    amax = max(amax, (unsigned)__shfl_xor((int)amax, 32, 64));
    if (hf == 0) most[wm][wn][n32] = amax;
    __syncthreads();
    const unsigned scale = fp8_block_scale(max(most[wm][0][n32], most[wm][1][n32]));
    __syncthreads();
    const float value = fp8_block_value(scale);
    // The codes in whole cache lines, as in store_rows (8193 rows, 5376 -> 14336 -> 5376: 0.5%). The
    // next row block writes there behind its own barriers.
    uint8_t *rows = (uint8_t *)scratch + CODE_ROWS + wm * 32 * CODE_ROW;
#pragma unroll
    for (int g = 0; g < 8; g += 2) {
        const auto s = __builtin_amdgcn_permlane32_swap(fp8_block_encode4(v + 4 * g, value),
                                                        fp8_block_encode4(v + 4 * g + 4, value), false, false);
        *reinterpret_cast<uint2 *>(rows + n32 * CODE_ROW + wn * 64 + hf * 8 + g * 8) = make_uint2(s[0], s[1]);
    }
    __syncthreads();
#pragma unroll
    for (unsigned r = wn * 16 + lane / 8, h = 0; h < 2; h++, r += 8) {
        const u32x4 o = *reinterpret_cast<const u32x4 *>(rows + r * CODE_ROW + lane % 8 * 16);
        if (row0 + r < a.m)
            __builtin_nontemporal_store(o, reinterpret_cast<u32x4 *>(a.out.codes + (size_t)(row0 + r) * a.out.stride + n0 / 2 +
                                                                     lane % 8 * 16));
    }
    if (row < a.m && wn == 0 && hf == 0) a.out.scales[fp8_block_scale_at(row, n0 / 256, a.out.groups)] = (uint8_t)scale;
}

// SPLIT: the tiles of the last, incomplete wave are shared over K.
template <int EPI, bool SPLIT, int TM>
__global__ __attribute__((amdgpu_flat_work_group_size(PIPE_T, PIPE_T), amdgpu_waves_per_eu(1, 1)))
void fp8_block_pipe(Fp8BlockGemmArgs a) {
    constexpr bool SWIGLU = EPI == EPI_SWIGLU;
    constexpr int NJ = TM / 64;               // row blocks of a wave
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const unsigned tid = threadIdx.x, lane = tid % 64, n32 = lane % 32, hf = lane / 32;
    const unsigned wave = __builtin_amdgcn_readfirstlane(tid / 64), wm = wave / 2, wn = wave % 2;
    unsigned ksteps = a.k / TK;
    TileShare t{};
    if constexpr (SPLIT) t = pipe_share(a, ksteps);
    else t.pid = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned k0 = t.first * TK;
    unsigned m0, n0;
    pipe_tile<TM>(a, t.pid, m0, n0);
    // Rows past M or N are past the resources' size and load zeros. SwiGLU: 32 gate rows and the
    // 32 up rows of the same columns alternate (loads of even and of odd number), so that a
    // lane's accumulator blocks hold both; a tile then makes 128 columns, one block of the
    // packed result.
    const unsigned xrows = min(a.m - m0, (unsigned)TM), wrows = SWIGLU ? 128u : min(a.n - n0, (unsigned)PIPE_N);
    const unsigned w0 = SWIGLU ? n0 / 2 : n0, w1 = SWIGLU ? n0 / 2 + a.n / 2 : n0;
    const i32x4 sx = asm_resource(a.x + (size_t)m0 * a.k + k0, xrows * a.k - k0);
    const i32x4 sw0 = asm_resource(a.w + (size_t)w0 * a.k + k0, wrows * a.k - k0);
    const i32x4 sw1 = asm_resource(a.w + (size_t)w1 * a.k + k0, wrows * a.k - k0);
    const unsigned blocks = (a.n + FP8_BLOCK - 1) / FP8_BLOCK;
    const unsigned g0 = t.first / QUAD;
    const i32x4 tx = asm_resource(a.xs + ((size_t)(m0 / 32) * a.groups + g0) * 128, (min((a.m + 31) / 32 - m0 / 32, TM / 32u) * a.groups - g0) * 128);
    const i32x4 tw = asm_resource(a.ws + (size_t)g0 * 128, ((blocks + 31) / 32 * a.groups - g0) * 128);
    const unsigned lrow = 8 * wave + lane / 8;
    unsigned ox[8], ow[8], oe[6];
#pragma unroll
    for (int b = 0; b < 8; b++) {
        ox[b] = (lrow + 32 * b) * a.k + swz(lrow, lane % 8) * 16;
        ow[b] = SWIGLU ? (lrow + 32 * (b / 2)) * a.k + swz(lrow, lane % 8) * 16 : ox[b];
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) oe[j] = (wm * NJ + j) * a.groups * 128 + n32 * 4;
    // A wave's 128 columns are one block of W; with SwiGLU the tile's gate rows are one, its up
    // rows another. A block past the end (a half-empty last tile) has no codes.
    const unsigned first_block = SWIGLU ? n0 / 256 : min(n0 / 128 + wn, blocks - 1);
    oe[4] = (unsigned)fp8_block_scale_at(first_block, 0, a.groups);
    oe[5] = SWIGLU ? (unsigned)fp8_block_scale_at(first_block + a.n / 256, 0, a.groups) : oe[4];
    const unsigned mb = __builtin_amdgcn_readfirstlane(wave * 1024);
    const unsigned kmax = __builtin_amdgcn_readfirstlane((ksteps - 1) * TK);
    const unsigned kgmax = __builtin_amdgcn_readfirstlane((ksteps - 1) / QUAD * 128);
    const unsigned kone = min(kmax, TK), ktwo = min(kmax, 2 * TK);
    unsigned kn = (TM == 256 ? 2 : 3) * TK, kc = 0, kg = 0, steps = __builtin_amdgcn_readfirstlane(ksteps);
    // Fragment bases in stage 0: row n32 of the wave's half, bytes 32 hf .. + 31 of substep
    // s, that is chunks 4 s + 2 hf and the next one.
    unsigned pw[2][2], px[2][2];
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const unsigned part = n32 * TK + swz(n32, 4 * s + 2 * hf + h) * 16;
            pw[s][h] = (TM == 256 ? 512 : 384) * TK + wn * 128 * TK + part;
            px[s][h] = wm * (TM / 2) * TK + part;
        }
    f32x16 c[4][NJ];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) c[i][j] = f32x16{};
    // Prologue: the first group's scales into set 0, tiles 0 and 1 into stages 0 and 1, substep
    // 0 of tile 0 into fragment set 0. The loop body is two groups of four tiles, left after
    // the last tile; loads past the end reload the last tile into a stage nobody reads again,
    // or the last group's scales.
    if constexpr (TM == 256)
    asm volatile(
        FB_SCALES(0)
        FB_FIRST(0, "0") FB_FIRST(1, "%[kone]")
        "s_waitcnt vmcnt(0)\n"
        "s_barrier\n"
        FB_RW(0, 0, 0, 0) FB_RW(0, 1, 0, 0) FB_RW(0, 2, 0, 0) FB_RW(0, 3, 0, 0)
        FB_RX(0, 0, 0, 0) FB_RX(0, 1, 0, 0) FB_RX(0, 2, 0, 0) FB_RX(0, 3, 0, 0)
        "s_waitcnt lgkmcnt(0)\n"
        "fb_loop_%=:\n"
        FB_QUAD(0, 1)
        FB_QUAD(1, 0)
        "s_branch fb_loop_%=\n"
        "fb_end_%=:\n"
        "s_waitcnt vmcnt(0) lgkmcnt(0)\n"
        // The last MFMAs' results are complete before the epilogue reads the accumulators
        // (hipcc does not see the MFMAs inside this block).
        "s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n"
        : FB_ACC4(0), FB_ACC4(1), FB_ACC4(2), FB_ACC4(3), [kc] "+s"(kc), [kn] "+s"(kn), [kg] "+s"(kg), [steps] "+s"(steps)
        : [sx] "s"(sx), [sw0] "s"(sw0), [sw1] "s"(sw1), [tx] "s"(tx), [tw] "s"(tw), [x0] "v"(ox[0]), [x1] "v"(ox[1]),
          [x2] "v"(ox[2]), [x3] "v"(ox[3]), [x4] "v"(ox[4]), [x5] "v"(ox[5]), [x6] "v"(ox[6]), [x7] "v"(ox[7]),
          [y0] "v"(ow[0]), [y1] "v"(ow[1]), [y2] "v"(ow[2]), [y3] "v"(ow[3]), [y4] "v"(ow[4]), [y5] "v"(ow[5]),
          [y6] "v"(ow[6]), [y7] "v"(ow[7]), [e0] "v"(oe[0]), [e1] "v"(oe[1]), [e2] "v"(oe[2]), [e3] "v"(oe[3]),
          [e4] "v"(oe[4]), [e5] "v"(oe[5]), [mb] "s"(mb), [kmax] "s"(kmax), [kgmax] "s"(kgmax), [kone] "s"(kone),
          [w00] "v"(pw[0][0]), [w01] "v"(pw[0][1]), [w10] "v"(pw[1][0]), [w11] "v"(pw[1][1]), [r00] "v"(px[0][0]),
          [r01] "v"(px[0][1]), [r10] "v"(px[1][0]), [r11] "v"(px[1][1])
        : "v64", "v65", "v66", "v67", "v68", "v69", FB_CL10(7), FB_CL10(8), FB_CL10(9), FB_CL10(10), FB_CL10(11),
          FB_CL10(12), FB_CL10(13), FB_CL10(14), FB_CL10(15), FB_CL10(16), FB_CL10(17), FB_CL10(18), FB_CL10(19),
          "v200", "v201", "v202", "v203", "m0", "scc", "memory");
    else {
    const unsigned pu[2][2] = {{pw[0][0] + 65536, pw[0][1] + 65536}, {pw[1][0] + 65536, pw[1][1] + 65536}};
    asm volatile(
        FH_SCALES(0)
        FH_FIRST(0, "0") FH_FIRST(1, "%[kone]") FH_FIRST(2, "%[ktwo]")
        "s_waitcnt vmcnt(24)\n"
        "s_barrier\n"
        FH_RW(0, 0, 0, 0) FH_RW(0, 1, 0, 0) FH_RW(0, 2, 0, 0) FH_RW(0, 3, 0, 0) FH_RX(0, 0, 0, 0) FH_RX(0, 1, 0, 0)
        "s_waitcnt lgkmcnt(0)\n"
        "fh_loop_%=:\n"
        FH_QUAD(0, 1, 2, 0, 1) FH_QUAD(1, 2, 0, 1, 0) FH_QUAD(2, 0, 1, 0, 1)
        FH_QUAD(0, 1, 2, 1, 0) FH_QUAD(1, 2, 0, 0, 1) FH_QUAD(2, 0, 1, 1, 0)
        "s_branch fh_loop_%=\n"
        "fh_end_%=:\n"
        "s_waitcnt vmcnt(0) lgkmcnt(0)\n"
        "s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n"
        : FH_ACC2(0), FH_ACC2(1), FH_ACC2(2), FH_ACC2(3), [kc] "+s"(kc), [kn] "+s"(kn), [kg] "+s"(kg), [steps] "+s"(steps)
        : [sx] "s"(sx), [sw0] "s"(sw0), [sw1] "s"(sw1), [tx] "s"(tx), [tw] "s"(tw), [x0] "v"(ox[0]), [x1] "v"(ox[1]),
          [x2] "v"(ox[2]), [x3] "v"(ox[3]), [y0] "v"(ow[0]), [y1] "v"(ow[1]), [y2] "v"(ow[2]), [y3] "v"(ow[3]),
          [y4] "v"(ow[4]), [y5] "v"(ow[5]), [y6] "v"(ow[6]), [y7] "v"(ow[7]), [e0] "v"(oe[0]), [e1] "v"(oe[1]),
          [e4] "v"(oe[4]), [e5] "v"(oe[5]), [mb] "s"(mb), [kmax] "s"(kmax), [kgmax] "s"(kgmax), [kone] "s"(kone),
          [ktwo] "s"(ktwo), [w00] "v"(pw[0][0]), [w01] "v"(pw[0][1]), [w10] "v"(pw[1][0]), [w11] "v"(pw[1][1]),
          [u00] "v"(pu[0][0]), [u01] "v"(pu[0][1]), [u10] "v"(pu[1][0]), [u11] "v"(pu[1][1]), [r00] "v"(px[0][0]),
          [r01] "v"(px[0][1]), [r10] "v"(px[1][0]), [r11] "v"(px[1][1])
        : "v64", "v65", "v66", "v67", "v68", "v69", FB_CL10(7), FB_CL10(8), FB_CL10(9), FB_CL10(10), FB_CL10(11),
          FB_CL10(12), FB_CL10(13), FB_CL10(14), FB_CL10(15), "v160", "v161", "v162", "v163", "v164", "v165", "v166",
          "v167", "m0", "scc", "memory");
    }

    // Block (i, j): lane holds output row m0 + TM / 2 wm + 32 j + n32.
    if (SPLIT && t.partial) {
        f32x4 *dst = reinterpret_cast<f32x4 *>(a.tile.part) +
                     ((size_t)t.tile * a.tile.split + t.share) * (TM * PIPE_N / 4) + tid;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            if (m0 + wm * (TM / 2) + j * 32 >= a.m) break;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                hold(c[i][j]);
#pragma unroll
                for (int g = 0; g < 4; g++)
                    dst[((j * 4 + i) * 4 + g) * 256] =
                        f32x4{c[i][j][4 * g], c[i][j][4 * g + 1], c[i][j][4 * g + 2], c[i][j][4 * g + 3]};
            }
        }
        return;
    }
    // Behind the last tile no wave reads its fragments any more once all have arrived here.
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
        for (int i = 0; i < 4; i++) hold(c[i][j]);
        pipe_epilogue<EPI>(a, m0 + wm * (TM / 2) + j * 32, n0, wm, wn, lane, c[0][j], c[1][j], c[2][j], c[3][j], lds);
    }
}

// The split tiles' shares added in order, and the epilogue. One workgroup per (tile, row block).
template <int EPI, int TM>
__global__ __launch_bounds__(PIPE_T) void fp8_block_pipe_reduce(Fp8BlockGemmArgs a) {
    constexpr unsigned NJ = TM / 64;
    __shared__ __attribute__((aligned(16))) uint8_t scratch[EPI == EPI_ANY ? ANY_LDS : EPI == EPI_SWIGLU ? CODE_ROWS + 2 * 32 * CODE_ROW : 4 * 32 * ROW_LDS<4>];
    const unsigned tile = blockIdx.x / NJ, j = blockIdx.x % NJ, tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    unsigned m0, n0;
    pipe_tile<TM>(a, split_tile(a.tile, tile), m0, n0);
    const unsigned row0 = m0 + wave / 2 * (TM / 2) + j * 32;
    const f32x4 *src = reinterpret_cast<const f32x4 *>(a.tile.part) + (size_t)tile * a.tile.split * (TM * PIPE_N / 4) +
                       j * 16 * 256 + tid;
    f32x16 c[4] = {};
    // A row block past M: no share was written.
    for (unsigned s = 0; row0 < a.m && s < a.tile.split; s++, src += TM * PIPE_N / 4)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const f32x4 v = src[(i * 4 + g) * 256];
#pragma unroll
                for (int e = 0; e < 4; e++) c[i][4 * g + e] += v[e];
            }
    pipe_epilogue<EPI>(a, row0, n0, wave / 2, wave % 2, lane, c[0], c[1], c[2], c[3], scratch);
}

// ---------------------------------------------------------------- tiles of 64 rows
// 64 x 256 outputs per workgroup, four waves of 64 x 64 and half as many products a tile again:
// four stages, X at 0, 8, 16 and 24 KB, W at 32, 64, 96 and 128 KB (all of a CU's LDS), loads
// four tiles ahead. Fragment set S in v[64 + 32 S ..], W block I at + 8 I, X block J at + 16 +
// 8 J; scale set Z in v[128 + 4 Z ..], X block J at + J, W at + 2 and + 3. Tile B of a group of
// four is in stage B. Bound by LDS, whose reads and writes take 1.6 times as long as the
// products, and by the memory's latency.
constexpr int MID_M = 64, MID_N = 256, MID_T = 256;
constexpr unsigned MID_LDS = 4 * (MID_M + MID_N) * TK;
constexpr int MID_GROUP = 4;

#define FQ_LX(ST, T) "s_add_u32 m0, %[mb], 8192*" #ST "+4096*" #T "\n"                                              \
    "buffer_load_dwordx4 %[x" #T "], %[sx], %[kc] offen lds\n"
#define FQ_LW(ST, T, R) "s_add_u32 m0, %[mb], 32768+32768*" #ST "+4096*" #T "\n"                                    \
    "buffer_load_dwordx4 %[y" #T "], %[sw" #R "], %[kc] offen lds\n"
#define FQ_SCALES(Z)                                                                                                \
    "buffer_load_dword v[128+4*" #Z "], %[e0], %[tx], %[kg] offen\n"                                                 \
    "buffer_load_dword v[128+4*" #Z "+1], %[e1], %[tx], %[kg] offen\n"                                               \
    "buffer_load_dword v[128+4*" #Z "+2], %[e2], %[tw], %[kg] offen\n"                                               \
    "buffer_load_dword v[128+4*" #Z "+3], %[e3], %[tw], %[kg] offen\n"                                               \
    "s_add_u32 %[kg], %[kg], 128\n"                                                                                 \
    "s_min_u32 %[kg], %[kg], %[kgmax]\n"
#define FQ_MFMA(S, Z, B, I, J)                                                                                      \
    "v_mfma_scale_f32_32x32x64_f8f6f4 %[c" #I #J "], v[64+32*" #S "+8*" #I ":64+32*" #S "+8*" #I "+7], "             \
    "v[64+32*" #S "+16+8*" #J ":64+32*" #S "+16+8*" #J "+7], %[c" #I #J "], v[128+4*" #Z "+2+" #I "], "              \
    "v[128+4*" #Z "+" #J "]" FB_SEL_##B
#define FQ_WAT_0(KS, H) "%[w" #KS #H "] offset:"
#define FQ_WAT_1(KS, H) "%[w" #KS #H "] offset:32768+"
#define FQ_WAT_2(KS, H) "%[u" #KS #H "] offset:"
#define FQ_WAT_3(KS, H) "%[u" #KS #H "] offset:32768+"
#define FQ_RW(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+32*" #T "+8*" #F ":64+32*" #T "+8*" #F "+3], " FQ_WAT_##ST(KS, 0) "4096*" #F "\n"              \
    "ds_read_b128 v[64+32*" #T "+8*" #F "+4:64+32*" #T "+8*" #F "+7], " FQ_WAT_##ST(KS, 1) "4096*" #F "\n"
#define FQ_RX(T, F, KS, ST)                                                                                         \
    "ds_read_b128 v[64+32*" #T "+16+8*" #F ":64+32*" #T "+16+8*" #F "+3], %[r" #KS "0] offset:8192*" #ST "+4096*" #F "\n" \
    "ds_read_b128 v[64+32*" #T "+16+8*" #F "+4:64+32*" #T "+16+8*" #F "+7], %[r" #KS "1] offset:8192*" #ST "+4096*" #F "\n"
#define FQ_SUB(S, Z, B, T, KS, ST, L0, L1, L2, L3)                                                                  \
    FQ_MFMA(S, Z, B, 0, 0) FQ_RW(T, 0, KS, ST) FQ_RX(T, 0, KS, ST) L0                                                \
    FQ_MFMA(S, Z, B, 0, 1) FQ_RX(T, 1, KS, ST) FQ_RW(T, 1, KS, ST) L1                                                \
    FQ_MFMA(S, Z, B, 1, 0) L2 FQ_MFMA(S, Z, B, 1, 1) L3
#define FQ_SUB_EXP(...) FQ_SUB(__VA_ARGS__)
#define FQ_NONE "", "", "", ""
#define FQ_LOADS(ST) FQ_LX(ST, 0) FQ_LW(ST, 0, 0), FQ_LX(ST, 1) FQ_LW(ST, 1, 1),                                      \
    FQ_LW(ST, 2, 0) FQ_LW(ST, 3, 1) FQ_LW(ST, 4, 0), FQ_LW(ST, 5, 1) FQ_LW(ST, 6, 0) FQ_LW(ST, 7, 1)
// The loads of the two tiles after the next (20, the youngest) stay in flight at the barrier.
#define FQ_TILE(ST, OT, Z, NEXT)                                                                                    \
    FQ_SUB_EXP(0, Z, ST, 1, 1, ST, FQ_NONE)                                                                          \
    "s_waitcnt vmcnt(20) lgkmcnt(0)\n"                                                                              \
    "s_barrier\n"                                                                                                   \
    "s_min_u32 %[kc], %[kn], %[kmax]\n"                                                                             \
    "s_add_u32 %[kn], %[kn], 128\n" NEXT                                                                            \
    FQ_SUB_EXP(1, Z, ST, 0, 0, OT, FQ_LOADS(ST))                                                                     \
    "s_waitcnt lgkmcnt(0)\n"                                                                                        \
    "s_sub_u32 %[steps], %[steps], 1\n"                                                                             \
    "s_cmp_eq_u32 %[steps], 0\n"                                                                                    \
    "s_cbranch_scc1 fq_end_%=\n"
#define FQ_QUAD(Z, OZ) FQ_TILE(0, 1, Z, FQ_SCALES(OZ)) FQ_TILE(1, 2, Z, "") FQ_TILE(2, 3, Z, "") FQ_TILE(3, 0, Z, "")
#define FQ_FIRST(ST, KC) "s_mov_b32 %[kc], " KC "\n" FQ_LX(ST, 0) FQ_LW(ST, 0, 0) FQ_LX(ST, 1) FQ_LW(ST, 1, 1)           \
    FQ_LW(ST, 2, 0) FQ_LW(ST, 3, 1) FQ_LW(ST, 4, 0) FQ_LW(ST, 5, 1) FQ_LW(ST, 6, 0) FQ_LW(ST, 7, 1)

__device__ inline void mid_tile(const Fp8BlockGemmArgs &a, unsigned pid, unsigned &m0, unsigned &n0) {
    unsigned tm, tn;
    band_tile((a.m + MID_M - 1) / MID_M, (a.n + MID_N - 1) / MID_N, MID_GROUP, pid, tm, tn);
    m0 = __builtin_amdgcn_readfirstlane(tm * MID_M);
    n0 = __builtin_amdgcn_readfirstlane(tn * MID_N);
}

// The epilogue of a wave's row block (32 rows from row0) and two column blocks from col0.
// SwiGLU: the four waves of a row meet in scratch (LDS) for the block's largest magnitude.
template <int EPI>
__device__ inline void mid_epilogue(const Fp8BlockGemmArgs &a, unsigned row0, unsigned n0, unsigned wn, unsigned lane,
                                    const f32x16 &c0, const f32x16 &c1, void *scratch) {
    const unsigned n32 = lane % 32, hf = lane / 32, row = row0 + n32;
    auto most = (unsigned(*)[32])scratch;
    if constexpr (EPI == EPI_PLAIN || EPI == EPI_BIAS) {
        store_rows<EPI, false, 2>(a, row0, n0 + wn * 64, lane, {&c0, &c1}, (uint8_t *)scratch + wn * 32 * ROW_LDS<2>);
        return;
    }
    if constexpr (EPI == EPI_ANY) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            store4<EPI>(a, row, n0 + wn * 64 + g * 8 + hf * 4, f32x4{c0[4 * g], c0[4 * g + 1], c0[4 * g + 2], c0[4 * g + 3]});
            store4<EPI>(a, row, n0 + wn * 64 + 32 + g * 8 + hf * 4, f32x4{c1[4 * g], c1[4 * g + 1], c1[4 * g + 2], c1[4 * g + 3]});
        }
        return;
    }
    float v[16];
    bool bad = false;
    float gate[16], up[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
        gate[e] = c0[e];
        up[e] = c1[e];
    }
    swiglu<16, true>(gate, up, v);
    unsigned amax = fp8_block_magnitude<16>(v, bad);
    if (bad && row < a.m) *a.out.fault = 1u;
    amax = max(amax, (unsigned)__shfl_xor((int)amax, 32, 64));
    if (hf == 0) most[wn][n32] = amax;
    __syncthreads();
    const unsigned scale = fp8_block_scale(max(max(most[0][n32], most[1][n32]), max(most[2][n32], most[3][n32])));
    __syncthreads();
    if (row >= a.m) return;
    const float value = fp8_block_value(scale);
    uint8_t *dst = a.out.codes + (size_t)row * a.out.stride + n0 / 2 + wn * 32 + hf * 4;
#pragma unroll
    for (int g = 0; g < 4; g++) *reinterpret_cast<unsigned *>(dst + g * 8) = fp8_block_encode4(v + 4 * g, value);
    if (wn == 0 && hf == 0) a.out.scales[fp8_block_scale_at(row, n0 / 256, a.out.groups)] = (uint8_t)scale;
}

template <int EPI, bool SPLIT>
__global__ __attribute__((amdgpu_flat_work_group_size(MID_T, MID_T), amdgpu_waves_per_eu(1, 1)))
void fp8_block_mid(Fp8BlockGemmArgs a) {
    constexpr bool SWIGLU = EPI == EPI_SWIGLU;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const unsigned tid = threadIdx.x, lane = tid % 64, n32 = lane % 32, hf = lane / 32;
    const unsigned wn = __builtin_amdgcn_readfirstlane(tid / 64);
    unsigned ksteps = a.k / TK;
    TileShare t{};
    if constexpr (SPLIT) t = pipe_share(a, ksteps);
    else t.pid = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned k0 = t.first * TK;
    unsigned m0, n0;
    mid_tile(a, t.pid, m0, n0);
    // As in fp8_block_pipe.
    const unsigned xrows = min(a.m - m0, (unsigned)MID_M), wrows = SWIGLU ? 128u : min(a.n - n0, (unsigned)MID_N);
    const unsigned w0 = SWIGLU ? n0 / 2 : n0, w1 = SWIGLU ? n0 / 2 + a.n / 2 : n0;
    const i32x4 sx = asm_resource(a.x + (size_t)m0 * a.k + k0, xrows * a.k - k0);
    const i32x4 sw0 = asm_resource(a.w + (size_t)w0 * a.k + k0, wrows * a.k - k0);
    const i32x4 sw1 = asm_resource(a.w + (size_t)w1 * a.k + k0, wrows * a.k - k0);
    const unsigned blocks = (a.n + FP8_BLOCK - 1) / FP8_BLOCK, g0 = t.first / QUAD;
    const i32x4 tx = asm_resource(a.xs + ((size_t)(m0 / 32) * a.groups + g0) * 128,
                                  (min((a.m + 31) / 32 - m0 / 32, MID_M / 32u) * a.groups - g0) * 128);
    const i32x4 tw = asm_resource(a.ws + (size_t)g0 * 128, ((blocks + 31) / 32 * a.groups - g0) * 128);
    const unsigned lrow = 8 * wn + lane / 8, part = swz(lrow, lane % 8) * 16;
    unsigned ow[8];
#pragma unroll
    for (int b = 0; b < 8; b++) ow[b] = (lrow + 32 * (SWIGLU ? b / 2 : b)) * a.k + part;
    const unsigned ox0 = lrow * a.k + part, ox1 = ox0 + 32 * a.k;
    const unsigned oe0 = n32 * 4, oe1 = a.groups * 128 + n32 * 4;
    // A wave's 64 columns are in one block of W; SwiGLU: 32 gate and 32 up columns.
    const unsigned first_block = SWIGLU ? n0 / 256 : min(n0 / 128 + wn / 2, blocks - 1);
    const unsigned oe2 = (unsigned)fp8_block_scale_at(first_block, 0, a.groups);
    const unsigned oe3 = SWIGLU ? (unsigned)fp8_block_scale_at(first_block + a.n / 256, 0, a.groups) : oe2;
    const unsigned mb = __builtin_amdgcn_readfirstlane(wn * 1024);
    const unsigned kmax = __builtin_amdgcn_readfirstlane((ksteps - 1) * TK);
    const unsigned kgmax = __builtin_amdgcn_readfirstlane((ksteps - 1) / QUAD * 128);
    const unsigned kone = min(kmax, TK), ktwo = min(kmax, 2 * TK), kthree = min(kmax, 3 * TK);
    unsigned kn = 4 * TK, kc = 0, kg = 0, steps = __builtin_amdgcn_readfirstlane(ksteps);
    unsigned pw[2][2], pu[2][2], px[2][2];
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            px[s][h] = n32 * TK + swz(n32, 4 * s + 2 * hf + h) * 16;
            pw[s][h] = 32768 + wn * 64 * TK + px[s][h];
            pu[s][h] = pw[s][h] + 65536;
        }
    f32x16 c[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) c[i][j] = f32x16{};
    asm volatile(
        FQ_SCALES(0)
        FQ_FIRST(0, "0") FQ_FIRST(1, "%[kone]") FQ_FIRST(2, "%[ktwo]") FQ_FIRST(3, "%[kthree]")
        "s_waitcnt vmcnt(30)\n"
        "s_barrier\n"
        FQ_RW(0, 0, 0, 0) FQ_RW(0, 1, 0, 0) FQ_RX(0, 0, 0, 0) FQ_RX(0, 1, 0, 0)
        "s_waitcnt lgkmcnt(0)\n"
        "fq_loop_%=:\n"
        FQ_QUAD(0, 1)
        FQ_QUAD(1, 0)
        "s_branch fq_loop_%=\n"
        "fq_end_%=:\n"
        "s_waitcnt vmcnt(0) lgkmcnt(0)\n"
        "s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n s_nop 7\n"
        : [c00] "+a"(c[0][0]), [c01] "+a"(c[0][1]), [c10] "+a"(c[1][0]), [c11] "+a"(c[1][1]), [kc] "+s"(kc), [kn] "+s"(kn),
          [kg] "+s"(kg), [steps] "+s"(steps)
        : [sx] "s"(sx), [sw0] "s"(sw0), [sw1] "s"(sw1), [tx] "s"(tx), [tw] "s"(tw), [x0] "v"(ox0), [x1] "v"(ox1),
          [y0] "v"(ow[0]), [y1] "v"(ow[1]), [y2] "v"(ow[2]), [y3] "v"(ow[3]), [y4] "v"(ow[4]), [y5] "v"(ow[5]),
          [y6] "v"(ow[6]), [y7] "v"(ow[7]), [e0] "v"(oe0), [e1] "v"(oe1), [e2] "v"(oe2), [e3] "v"(oe3), [mb] "s"(mb),
          [kmax] "s"(kmax), [kgmax] "s"(kgmax), [kone] "s"(kone), [ktwo] "s"(ktwo), [kthree] "s"(kthree),
          [w00] "v"(pw[0][0]), [w01] "v"(pw[0][1]), [w10] "v"(pw[1][0]), [w11] "v"(pw[1][1]), [u00] "v"(pu[0][0]),
          [u01] "v"(pu[0][1]), [u10] "v"(pu[1][0]), [u11] "v"(pu[1][1]), [r00] "v"(px[0][0]), [r01] "v"(px[0][1]),
          [r10] "v"(px[1][0]), [r11] "v"(px[1][1])
        : "v64", "v65", "v66", "v67", "v68", "v69", FB_CL10(7), FB_CL10(8), FB_CL10(9), FB_CL10(10), FB_CL10(11),
          FB_CL10(12), "v130", "v131", "v132", "v133", "v134", "v135", "m0", "scc", "memory");

    // Block (i, j): lane holds output row m0 + 32 j + n32.
    if (SPLIT && t.partial) {
        f32x4 *dst = reinterpret_cast<f32x4 *>(a.tile.part) +
                     ((size_t)t.tile * a.tile.split + t.share) * (MID_M * MID_N / 4) + tid;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (m0 + j * 32 >= a.m) break;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                hold(c[i][j]);
#pragma unroll
                for (int g = 0; g < 4; g++)
                    dst[((j * 2 + i) * 4 + g) * MID_T] =
                        f32x4{c[i][j][4 * g], c[i][j][4 * g + 1], c[i][j][4 * g + 2], c[i][j][4 * g + 3]};
            }
        }
        return;
    }
    if constexpr (EPI != EPI_ANY) __syncthreads();     // all have read their last fragments
#pragma unroll
    for (int j = 0; j < 2; j++) {
        hold(c[0][j]);
        hold(c[1][j]);
        mid_epilogue<EPI>(a, m0 + j * 32, n0, wn, lane, c[0][j], c[1][j], lds);
    }
}

// The split tiles' shares added in order, and the epilogue. One workgroup per (tile, row block).
template <int EPI>
__global__ __launch_bounds__(MID_T) void fp8_block_mid_reduce(Fp8BlockGemmArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t scratch[EPI == EPI_SWIGLU ? 512 : EPI == EPI_ANY ? 16 : 4 * 32 * ROW_LDS<2>];
    const unsigned tile = blockIdx.x / 2, j = blockIdx.x % 2, tid = threadIdx.x;
    unsigned m0, n0;
    mid_tile(a, split_tile(a.tile, tile), m0, n0);
    const unsigned row0 = m0 + j * 32;
    if (row0 >= a.m) return;       // no share was written
    const f32x4 *src = reinterpret_cast<const f32x4 *>(a.tile.part) + (size_t)tile * a.tile.split * (MID_M * MID_N / 4) +
                       j * 8 * MID_T + tid;
    f32x16 c[2] = {};
#pragma unroll 2
    for (unsigned s = 0; s < a.tile.split; s++, src += MID_M * MID_N / 4)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const f32x4 v = src[(i * 4 + g) * MID_T];
#pragma unroll
                for (int e = 0; e < 4; e++) c[i][4 * g + e] += v[e];
            }
    mid_epilogue<EPI>(a, row0, n0, tid / 64, tid % 64, c[0], c[1], scratch);
}

template <int EPI> int launch_mid(h3_gpu *g, Fp8BlockGemmArgs a, unsigned split) {
    static bool configured = false;
    if (!configured) {
        for (const void *kernel : {(const void *)fp8_block_mid<EPI, false>, (const void *)fp8_block_mid<EPI, true>})
            if (!h3_hip_check(g, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, MID_LDS),
                              "FP8 block GEMM shared memory"))
                return 0;
        configured = true;
    }
    const unsigned tiles = (a.m + MID_M - 1) / MID_M * ((a.n + MID_N - 1) / MID_N), quads = (a.k / TK + QUAD - 1) / QUAD;
    a.tile = split_last_wave(g, tiles, split, quads, MID_M * MID_N);
    const unsigned rest = tiles - a.tile.full;
    h3_note_kernel(g, "fp8_block_mid", MID_M, a.tile.split);
    hipEvent_t timing = h3_kernel_timing_begin(g);
    if (!rest) {
        hipLaunchKernelGGL((fp8_block_mid<EPI, false>), dim3(tiles), dim3(MID_T), MID_LDS, g->compute, a);
    } else {
        hipLaunchKernelGGL((fp8_block_mid<EPI, true>), dim3(a.tile.full + rest * a.tile.split), dim3(MID_T), MID_LDS, g->compute, a);
        if (h3_launch_status(g, "FP8 block GEMM"))
            hipLaunchKernelGGL(fp8_block_mid_reduce<EPI>, dim3(rest * 2), dim3(MID_T), 0, g->compute, a);
    }
    h3_kernel_timing_end(g, timing);
    return h3_launch_status(g, "FP8 block GEMM");
}

template <int EPI, int TM> int launch_pipe(h3_gpu *g, Fp8BlockGemmArgs a, unsigned split) {
    constexpr unsigned shared = pipe_lds<TM>();
    static bool configured = false;
    if (!configured) {
        for (const void *kernel : {(const void *)fp8_block_pipe<EPI, false, TM>, (const void *)fp8_block_pipe<EPI, true, TM>})
            if (!h3_hip_check(g, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, shared),
                              "FP8 block GEMM shared memory"))
                return 0;
        configured = true;
    }
    const unsigned tiles = (a.m + TM - 1) / TM * ((a.n + PIPE_N - 1) / PIPE_N), quads = (a.k / TK + QUAD - 1) / QUAD;
    a.tile = split_last_wave(g, tiles, split, quads, TM * PIPE_N);
    const unsigned rest = tiles - a.tile.full;
    h3_note_kernel(g, "fp8_block_pipe", TM, a.tile.split);
    hipEvent_t timing = h3_kernel_timing_begin(g);
    if (!rest) {
        hipLaunchKernelGGL((fp8_block_pipe<EPI, false, TM>), dim3(tiles), dim3(PIPE_T), shared, g->compute, a);
    } else {
        hipLaunchKernelGGL((fp8_block_pipe<EPI, true, TM>), dim3(a.tile.full + rest * a.tile.split), dim3(PIPE_T), shared,
                           g->compute, a);
        if (h3_launch_status(g, "FP8 block GEMM"))
            hipLaunchKernelGGL((fp8_block_pipe_reduce<EPI, TM>), dim3(rest * (TM / 64)), dim3(PIPE_T), 0, g->compute, a);
    }
    h3_kernel_timing_end(g, timing);
    return h3_launch_status(g, "FP8 block GEMM");
}

// ---------------------------------------------------------------- choice
// The kernel whose modelled time is least. Tiles by gemm_last_wave in units of four K steps of
// 128. Few rows: the workgroups of the busiest CU by their K steps. Rates fitted to the measured
// times of all of them, the tiles in one to nine shares, at 259 projections of 1 to 8000 rows
// (K 256 to 14336, N 300 to 32256; weights that rotate through more than the last cache holds);
// the choice is 0.9% slower than the best of them in the mean. Measured, in us, the runner-up in
// brackets: 1 row, 7168 -> 5376: 9.7 (tiles of 64 rows in 4 shares 15.7); 32 rows, 5376 -> 21504:
// tiles of 64 in 2 shares 28.8 (128 rows in 2 shares 30.5); 640 rows, 13824 -> 5120: 128 rows in 2
// shares 50.5 (64 rows 57.6); 1024 rows, 7168 -> 5376: 128 rows 38.7 (256 in 2 shares 49.4); 1500
// rows, 5376 -> 21504: 256 rows 146.4 (128 rows 153.8).
// A launch has fewer than 2^32 threads: kernels whose grid would have more are no candidates.
constexpr uint64_t MAX_THREADS = 0xffffffffu;
struct Choice {
    float us;
    unsigned rows, split;     // tile rows (64, 128, 256) and shares; or
    unsigned rb, nb;          // few rows: row and column blocks (rb 0: tiles)
};
// Few rows: us of a step, [row blocks - 1][column blocks 2, 4], and the busiest CU's workgroups;
// of a byte of x that such a CU reads (from L2). None is faster than the weight's reads: 6.6 TB/s
// for few rows, beside their launch, 5.1 for tiles.
constexpr float STREAM_LAUNCH = 3.26f, STREAM_BYTE = 1.52e-7f, STREAM_X = 2.05e-5f, TILE_BYTE = 1.95e-7f;
constexpr float STREAM_STEP[3][2] = {{.14f, .26f}, {.17f, .32f}, {.27f, 0.f}};
Choice choose(const h3_gpu *g, const Fp8BlockGemmArgs &a, bool few, bool tiled = true) {
    static constexpr GemmRates RATES[3] = {{2.44f, 1.82f, .654f, .15f, 1.67f, .0881f, 1.12f},
                                           {4.02f, 1.99f, 1.82f, .3f, 3.61f, .0557f, 1.02f},
                                           {7.38f, 3.62f, 4.18f, .3f, 8.77f, .0346f, 1.f}};
    static constexpr float LAUNCH[3] = {2.77f, 3.54f, 0.f};
    const float reads = (float)a.n * a.k;
    const unsigned steps = a.k / TK;
    Choice best{3.4e38f, 0, 1, 0, 0};
    for (unsigned i = 0; tiled && i < 3; i++) {
        const unsigned rows = 64u << i, units = (steps + QUAD - 1) / QUAD;
        const uint64_t tiles = ((uint64_t)a.m + rows - 1) / rows * (((uint64_t)a.n + 255) / 256);
        if ((tiles + 2 * g->cus) * 256 > MAX_THREADS) continue;     // and the shares of a last wave
        const GemmPlan p = gemm_last_wave(g, (unsigned)tiles, units, RATES[i], rows / 256.f);
        const float us = (std::max(p.us, reads * TILE_BYTE) + LAUNCH[i]) * (p.split > 1 ? 1.02f : 1.f);
        if (us < best.us) best = {us, rows, p.split, 0, 0};
    }
    if (!few) return best;
    for (unsigned rb = 1; rb <= 3; rb++)
        for (unsigned nb = 2; nb <= (rb < 3 ? 4u : 2u); nb += 2) {
            const float rounds = stream_rounds(g, a, rb, nb);
            if (stream_groups(a, rb, nb) * (rb == 1 && nb == 2 ? 512 : 256) > MAX_THREADS) continue;
            const float us = STREAM_LAUNCH + std::max(rounds * steps * STREAM_STEP[rb - 1][nb / 4], reads * STREAM_BYTE) +
                             rounds * std::min(a.m, 16 * rb) * a.k * STREAM_X;
            if (us < best.us) best = {us, 0, 1, rb, nb};
        }
    return best;
}

// Whether a projection of few rows packs its BF16 input itself: a launch is 2.5 us, packing a
// step and row block 0.07 us beside the loads of a CU's one workgroup, 0.3 us where several
// share its VALU.
bool packs(const h3_gpu *g, const Fp8BlockGemmArgs &a, const Choice &c) {
    if (!c.rb) return false;
    const float rounds = stream_rounds(g, a, c.rb, c.nb);
    return rounds * (a.k / TK) * c.rb * (rounds > 1.f ? .3f : .07f) < 2.5f;
}

template <int EPI> int run(h3_gpu *g, const Fp8BlockGemmArgs &a) {
    // SwiGLU is an epilogue of tiles only; the sums are asked for where few rows' kernels are faster.
    constexpr bool few = EPI != EPI_SWIGLU, tiles = EPI != EPI_SUMS;
    const Choice c = choose(g, a, few, tiles);
    if (a.m > FP8_BLOCK_ROWS || (!c.rb && !c.rows))
        return h3_set_error(g, "FP8 block projection: %u rows by %u columns are too many for one call", a.m, a.n);
    if constexpr (few)
        if (c.rb) return a.xb ? launch_stream<EPI, true>(g, a, c.rb, c.nb) : launch_stream<EPI, false>(g, a, c.rb, c.nb);
    if constexpr (tiles) {
        if (a.xb) return h3_set_error(g, "FP8 block projection: %u rows of BF16 are to be packed first", a.m);
        return c.rows == 256   ? launch_pipe<EPI, 256>(g, a, c.split)
               : c.rows == 128 ? launch_pipe<EPI, 128>(g, a, c.split)
                               : launch_mid<EPI>(g, a, c.split);
    }
    return 0;
}

}  // namespace

bool h3_gemm_fp8_block_packs(const h3_gpu *g, const Fp8BlockGemmArgs &a) { return packs(g, a, choose(g, a, !a.swiglu)); }

// Without it the product goes through memory in FP32 and another launch packs it.
bool h3_gemm_fp8_block_fuses(const h3_gpu *g, uint32_t m, uint32_t k, uint32_t hidden) {
    Fp8BlockGemmArgs a{};
    a.m = m; a.n = 2 * hidden; a.k = (k + TK - 1) / TK * TK;
    return choose(g, a, false).us <= choose(g, a, true).us + 4.f + (float)m * hidden * 4e-6f;
}

int h3_gemm_fp8_block(h3_gpu *g, const Fp8BlockGemmArgs &a) {
    switch (epilogue_of(a)) {
    case EPI_PLAIN: return run<EPI_PLAIN>(g, a);
    case EPI_BIAS: return run<EPI_BIAS>(g, a);
    case EPI_SWIGLU: return run<EPI_SWIGLU>(g, a);
    case EPI_SUMS: return run<EPI_SUMS>(g, a);
    default: return run<EPI_ANY>(g, a);
    }
}
