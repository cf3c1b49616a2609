// Block-scaled FP8: the packed matrix, its encoding on the device, and the projection
// kernels' arguments (fp8_block.hip, gemm_fp8_block.hip, elementwise.hip).
//
// A matrix [rows, columns] is E4M3 codes in rows of `stride` bytes (columns rounded up to
// 128, the rest zero) and one E8M0 scale byte e + 127, value 2^e, per block of 128: an
// activation's block (tile 1) is 128 columns of one row, a weight's (tile 128) 128 rows by
// 128 columns. Scales lie as the products read them, lanes being rows: 32 scale rows by four
// blocks are 128 bytes, a dword of four blocks for each row; the `groups` fours of a row
// follow each other, then come the next 32 rows. (As rows of bytes, each lane's dword is in a
// cache line of its own: a quarter more traffic from L2 than the codes', and 2.5% of the time
// of a projection of 18225 rows, 5376 -> 28672.)
//
// Why powers of two: E4M3 is a floating-point type, so a scale's mantissa would not make its
// codes more exact, only extend their range below by less than one binade, while
// v_mfma_scale takes a power of two per row without a further instruction (an FP32 scale is
// an FMA per sum and block, half as many VALU cycles as the products take). x / 2^e is exact,
// so a code has one rounding.
#pragma once
#include "common.h"
#include "gemm.h"

constexpr uint32_t FP8_BLOCK = 128;
// Least exponent of a scale: blocks below 448 * 2^-64 lose their small values, and products
// of two scales stay in FP32's range.
constexpr int FP8_BLOCK_LEAST = -64;
// 256 rows of codes have 32-bit offsets.
constexpr uint32_t FP8_BLOCK_COLUMNS = (1u << 24) - FP8_BLOCK;
// Most rows of one projection launch: its tile numbers are computed in 32 bits.
constexpr uint32_t FP8_BLOCK_ROWS = 1u << 22;

struct Fp8BlockLayout {
    size_t stride, scales, groups, bytes;
};
inline Fp8BlockLayout fp8_block_layout(uint32_t rows, uint32_t columns, uint32_t tile) {
    const size_t blocks = (columns + FP8_BLOCK - 1) / FP8_BLOCK;
    Fp8BlockLayout l;
    l.stride = blocks * FP8_BLOCK;
    l.scales = ((size_t)rows * l.stride + 255) & ~(size_t)255;
    l.groups = (blocks + 3) / 4;
    l.bytes = l.scales + (((size_t)rows + tile - 1) / tile + 31) / 32 * l.groups * 128;
    return l;
}

// Byte of (scale row, block).
__host__ __device__ inline size_t fp8_block_scale_at(unsigned row, unsigned block, unsigned groups) {
    return ((size_t)(row / 32) * groups + block / 4) * 128 + row % 32 * 4 + block % 4;
}

// Where a packing kernel writes: row r's codes at codes + r * stride.
struct Fp8BlockRows {
    uint8_t *codes, *scales;
    unsigned stride, groups;
    unsigned *fault;      // set where a value is not finite
};

#if defined(__HIPCC__)
// Largest magnitude of N values as its bits, whose order is that of the values. Values that are
// not finite set bad and count as zero; they are looked for in the maximum only, above all of
// which they are. (The opaque step keeps the compiler, which assumes that no value is NaN, from
// folding the test.)
template <int N> __device__ inline unsigned fp8_block_magnitude(const float *v, bool &bad) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < N; e++) m = max(m, __builtin_bit_cast(unsigned, v[e]) & 0x7fffffffu);
    asm("" : "+v"(m));
    if (m >= 0x7f800000u) {
        bad = true;
        m = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const unsigned u = __builtin_bit_cast(unsigned, v[e]) & 0x7fffffffu;
            m = max(m, u >= 0x7f800000u ? 0u : u);
        }
    }
    return m;
}
// Scale byte of a block whose largest magnitude has these bits: the least e >= -64 with
// amax <= 448 * 2^e. 448 = 1.75 * 2^8, so e = exponent - 8, one more if the mantissa is
// above 1.75.
__device__ inline unsigned fp8_block_scale(unsigned amax) {
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)max(e, FP8_BLOCK_LEAST + 127);
}
// The scale's value, for the encoding.
__device__ inline float fp8_block_value(unsigned scale) { return __builtin_bit_cast(float, scale << 23); }
// Four codes of v / 2^e: round to nearest even; |v| <= 448 * 2^e.
__device__ inline unsigned fp8_block_encode4(const float *v, float value) {
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    i16x2 w = {};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[0], v[1], value, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[2], v[3], value, true);
    return __builtin_bit_cast(unsigned, w);
}
// Largest of `lanes` neighbouring lanes (a power of two up to 64).
template <int LANES> __device__ inline unsigned lanes_max(unsigned v) {
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 64));
    return v;
}
// silu(gate) * up = gate / (1 + exp(-gate)) * up in FP32, each step within about a unit in
// the last place, because a code flips where the value crosses a midpoint: exp(-gate) as 2^hi
// (1 + lo ln 2) with the product's rounding error in lo, and the reciprocal with a Newton step.
// For gates from SWIGLU_LEAST on; below, the reciprocal leaves FP32's normal range.
constexpr float SWIGLU_L = 1.4426950408889634f, SWIGLU_L_LOW = 1.9259629911266175e-8f, SWIGLU_LN2 = 0.6931471805599453f;
constexpr float SWIGLU_LEAST = -87.f;
__device__ inline float swiglu_exact(float gate, float up) {
    const float x = __builtin_amdgcn_fmed3f(gate, SWIGLU_LEAST, 128.f);       // exp(-128) is nothing beside 1
    const float hi = -x * SWIGLU_L, lo = -fmaf(x, SWIGLU_L, hi) - x * SWIGLU_L_LOW;
    const float e = __builtin_amdgcn_exp2f(hi), d = 1.f + fmaf(e, lo * SWIGLU_LN2, e);
    const float r = __builtin_amdgcn_rcpf(d);
    return gate * fmaf(fmaf(-d, r, 1.f), r, r) * up;
}
// The same for a projection's sums, whose own error (1.5e-5, the matrix core's additions) is
// far above what the two differ by, |gate| 2^-24: half the instructions, which nothing hides in
// an epilogue.
__device__ inline float swiglu_of_sums(float gate, float up) {
    return gate * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(gate * -SWIGLU_L)) * up;
}
// Gates below SWIGLU_LEAST, where 1 + exp(gate) is 1: gate exp(gate) up, the exponential 2^96 times
// as large and up 2^-96 times, so that both stay in FP32's normal range while their product with a
// large up is one. Below -153 it is zero: less than 2e-26 for any up, of which the least scale
// (2^-64) leaves nothing (not a number where the gate is infinite).
__device__ inline float swiglu_low(float gate, float up) {
    const float x = fmaxf(gate, -153.f), hi = x * SWIGLU_L, lo = fmaf(x, SWIGLU_L, -hi) + x * SWIGLU_L_LOW;
    const float e = __builtin_amdgcn_exp2f(hi + 96.f);
    return gate * (gate < -153.f ? 0.f : fmaf(e, lo * SWIGLU_LN2, e)) * (up * 0x1p-96f);
}
// N values v of gates and ups. Gates that are so low are rare: a branch for all of a lane's (their
// cases within the formulas above: 1% of an MLP of 8193 rows, 5376 -> 14336 -> 5376, and 5% of
// SwiGLU of 729 rows of 14336). Of sums, one branch behind all (one for each value: 1.5% of that
// MLP); else one for each, for the registers (SwiGLU of 8193 rows 175 us, with one 176.6).
template <int N, bool SUMS> __device__ inline void swiglu(const float *gate, const float *up, float *v) {
    float least = gate[0];
#pragma unroll
    for (int e = 1; e < N; e++) least = fminf(least, gate[e]);
    const bool low = least < SWIGLU_LEAST;
#pragma unroll
    for (int e = 0; e < N; e++) {
        v[e] = SUMS ? swiglu_of_sums(gate[e], up[e]) : swiglu_exact(gate[e], up[e]);
        if (!SUMS && low) v[e] = gate[e] < SWIGLU_LEAST ? swiglu_low(gate[e], up[e]) : v[e];
    }
    if (SUMS && low)
#pragma unroll
        for (int e = 0; e < N; e++)
            if (gate[e] < SWIGLU_LEAST) v[e] = swiglu_low(gate[e], up[e]);
}
#endif

// y = bf16(x . w^T + bias) and its variants (h3_gemm_fp8_block).
struct Fp8BlockGemmArgs {
    uint16_t *y;                // [m, n], or
    float *y32;                 // the sums as they are [m, n], or, with swiglu,
    Fp8BlockRows out;           // silu(gate) * up packed [m, n / 2]: w holds gate rows, then up rows
    const uint16_t *bias;       // [n], y only
    const uint8_t *x, *w;       // codes, rows of k bytes (a multiple of 128)
    const uint16_t *xb;         // BF16 rows of `columns` values instead of x and xs, only where
    unsigned columns;           // h3_gemm_fp8_block_packs; a value that is not finite sets fault
    unsigned *fault;
    const uint8_t *xs, *ws;     // scales; a scale row of w per 128 rows
    unsigned m, n, k, groups;
    bool swiglu;                // n / 2 a multiple of 128
    TileSplit tile;             // set by the kernels' launchers
};
int h3_gemm_fp8_block(h3_gpu *g, const Fp8BlockGemmArgs &a);
// Whether the projection would better pack a BF16 input itself than read a packed one (the
// same result bit for bit).
bool h3_gemm_fp8_block_packs(const h3_gpu *g, const Fp8BlockGemmArgs &a);
// Whether the SwiGLU variant is faster as one launch than as y32 and h3_launch_swiglu_fp8_block.
bool h3_gemm_fp8_block_fuses(const h3_gpu *g, uint32_t m, uint32_t k, uint32_t hidden);
// Packs silu(gate) * up of FP32 or BF16 rows [rows, 2 * width].
int h3_launch_swiglu_fp8_block(h3_gpu *g, Fp8BlockRows out, const void *fused, bool f32, uint32_t rows, uint32_t width);

// Entry-point helpers (fp8_block.hip): whether t is a packed matrix of this context with this
// tile, at least `rows` rows (tile 1; a weight: exactly) and `columns` columns, else the error.
int h3_require_fp8_block(h3_gpu *g, const h3_gpu_tensor *t, uint32_t tile, uint32_t rows, uint32_t columns,
                         const char *name);
Fp8BlockRows h3_fp8_block_rows(h3_gpu *g, const h3_gpu_tensor *t);
// A projection whose weight is packed in blocks and its input BF16 (packed here) or packed.
int h3_fp8_block_linear(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w,
                        const h3_gpu_tensor *bias, uint32_t rows, uint32_t k, uint32_t n);
int h3_fp8_block_mlp(h3_gpu *g, h3_gpu_tensor *out, const h3_gpu_tensor *in, const h3_gpu_tensor *w1,
                     const h3_gpu_tensor *w2, uint32_t rows, uint32_t k, uint32_t hidden, uint32_t n);
