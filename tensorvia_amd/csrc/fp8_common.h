// Shared pieces of the 8-bit floating-point layer: the number format, block scales, loads of short rows
// and the lane reductions.
//
// Format: OCP e4m3 codes (largest value 448) and one fp32 scale per block of 128 elements of a row
// (activations) or 128 x 128 elements (weights):
//     scale = max(max|x| / 448, 2^-126),   code = e4m3(x / scale), rounded to nearest even.
// The largest |x| maps to 448: no clamp is needed.  The floor of 2^-126 keeps 1 / scale finite in an all-zero block.
#pragma once
#include "tv_kernels.h"

namespace tvk {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

constexpr float kFp8Max = 448.0f;
constexpr float kFp8MinScale = 1.17549435e-38f; // 2^-126
constexpr unsigned kAbsMask = 0x7fffffffu;

// Magnitudes are compared as the integers of their bit patterns: the order of the magnitudes, with
// infinity above every number and NaN above infinity, so a NaN in a block reaches its scale.
__device__ inline unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & kAbsMask; }
__device__ inline unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }

// Scale of a block whose largest magnitude has these bits, and the factor of its codes in two parts: x * (hi + lo) is 448 x / max|x|
// to the last bit of fp32.  16-bit inputs often fall on the middle between two codes (448 x / max|x| = 232, say), which x times a
// rounded 1 / scale misses to either side: the error of bf16 codes is twice as large.  NaN stays NaN (the comparison is false);
// with an infinity the factor is 0, and only infinities give NaN.
struct Fp8Block {
    float scale, hi, lo;
    __device__ inline float operator()(float x) const { return __builtin_fmaf(x, hi, x * lo); }
};
__device__ inline Fp8Block fp8_block(unsigned amax) {
    const float a = __builtin_bit_cast(float, amax), floor = kFp8Max * kFp8MinScale, m = a < floor ? floor : a;
    Fp8Block f;
    f.scale = m / kFp8Max;
    f.hi = kFp8Max / m;
    f.lo = amax < 0x7f800000u ? __builtin_fmaf(-f.hi, m, kFp8Max) * (f.hi * (1.0f / kFp8Max)) : 0.0f;
    return f;
}

// Four codes of four values already divided by their scale.
__device__ inline unsigned cvt4_fp8(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
    return (unsigned)v;
}

// Lane permutations inside a row of 16 lanes (one DPP move each): row_ror:N rotates the row.
template <int N> __device__ inline unsigned row_ror(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 | N, 0xf, 0xf, true);
}
// Largest of 16 lanes' values, in all 16 lanes.
__device__ inline unsigned row16_max(unsigned x) {
    x = umax(x, row_ror<8>(x));
    x = umax(x, row_ror<4>(x));
    x = umax(x, row_ror<2>(x));
    return umax(x, row_ror<1>(x));
}
// Sum over a wave, in all lanes.
__device__ inline float wave_sum(float x) {
    x += __builtin_bit_cast(float, row_ror<8>(__builtin_bit_cast(unsigned, x)));
    x += __builtin_bit_cast(float, row_ror<4>(__builtin_bit_cast(unsigned, x)));
    x += __builtin_bit_cast(float, row_ror<2>(__builtin_bit_cast(unsigned, x)));
    x += __builtin_bit_cast(float, row_ror<1>(__builtin_bit_cast(unsigned, x)));
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

__device__ inline f32x4 mfma_fp8(const i32x8& w, const i32x8& a) {
    // Zero scale operands select the instruction without block exponents.
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}

// The same block sum with exact products and fp32 accumulation, for fp32 results.  The fp8 instructions align the products of 8 codes of
// a lane at a time and cut each, toward zero, to a multiple of 2^-13 of the largest one's power of two (looked at with one
// large and one small product; between the groups of 8 the sums keep fp32's bits).  On random codes that is 1.5e-5 of
// the block's sum, 16x16x128 and 16x16x32 alike; where one value of a row is 30, 100 or 448 times the others 3e-5, 5e-5
// and 6e-5.  A result rounded to 16 bits does not show it; an fp32 one would.  e4m3 values are exact in bf16, whose instruction
// accumulates in fp32 (9e-9), at half the rate.
// Codes 8 q to 8 q + 7 of a lane's 32, as bf16.
__device__ inline bf16x8 exact_codes(const i32x8& x, int q) {
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 pair;
    pair p[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        p[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q + j], 1.0f, false);
        p[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q + j], 1.0f, true);
    }
    return __builtin_bit_cast(bf16x8, p);
}
__device__ inline f32x4 mfma_fp8_exact(const i32x8& w, const i32x8& a) {
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(exact_codes(w, q), exact_codes(a, q), acc, 0, 0, 0);
    return acc;
}

// Elements k to k + 7 of a row of K, as floats with zeros past its end.  Any alignment: the 16-byte copies compile to unaligned
// vector loads.  The lanes at the end load the row's last eight elements and shift them down at their use, so that no lane
// takes a branch around a load, and several are on their way before the first is used (element by element the norm of 8192 rows of
// 4092 took 89 us, now 60; of 4096 58).
// SHORT: rows of less than eight elements (in one type with the others, the vector loads came apart: 20 -> 35 us for [8192,4096]).
template <typename T, bool SHORT = false> struct Eight {
    T e[8];
    __device__ inline void load(const T* row, int64_t k, int64_t K) {
        if constexpr (SHORT) {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = row[k + i < K ? k + i : 0];
        } else {
            __builtin_memcpy(e, row + (k < K - 8 ? k : K - 8), sizeof(e));
        }
    }
    __device__ inline void get(int64_t k, int64_t K, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)e[i];
        if constexpr (SHORT) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < K ? v[i] : 0.0f;
        } else if (k + 8 > K) {
            const int s = k < K ? (int)(k + 8 - K) : 8;
#pragma unroll
            for (int b = 8; b > 0; b >>= 1)
                if (s & b)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = i + b < 8 ? v[(i + b) & 7] : 0.0f;
        }
    }
};
template <typename T> __device__ inline void store8(T* p, int64_t n, const float (&v)[8]) {
    if (n >= 8) {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (T)v[i];
        __builtin_memcpy(p, e, sizeof(e));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}
__device__ inline void store_codes8(uint8_t* p, int64_t n, const float (&v)[8], const Fp8Block& f) {
    const unsigned lo = cvt4_fp8(f(v[0]), f(v[1]), f(v[2]), f(v[3]));
    const unsigned hi = cvt4_fp8(f(v[4]), f(v[5]), f(v[6]), f(v[7]));
    if (n >= 8) {
        const uint2 w = {lo, hi};
        __builtin_memcpy(p, &w, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// Most workgroups these launchers start (grid x block stays below 2^32 threads); kernels loop where there is more work, or
// are launched again.
constexpr int64_t kMaxGrid = 1 << 20;

// How the rows of a product's operands lie: whole 16-byte chunks at 16-byte aligned addresses, or anything.  A lane holds 32
// codes of a block of 128: two chunks of 16, 64 apart, of aligned rows (an instruction then reads 64 bytes of each of 16
// rows), 32 in a row of others.
enum Fp8Rows { FP8_ANY = 0, FP8_ALIGNED = 1 };
template <int ROWS> constexpr int kLaneStep = ROWS == FP8_ALIGNED ? 16 : 32;  // bytes from lane group to lane group
template <int ROWS> constexpr int kSecondHalf = ROWS == FP8_ALIGNED ? 64 : 16; // a lane's second 16 bytes after its first

// A lane's 32 codes on their way: raw words, put in place at their use.  Loads of 16 bytes that are not at a multiple of 4
// bytes take two and a half times as long (bf16 [1,4095]x[11008,4095]: 25.5 us, 11.6 with rows of 4100), so other rows are
// read as the words that hold them and shifted.
template <int ROWS> struct LaneCodes {
    u32x4 lo, hi;
    unsigned next; // FP8_ANY: the word behind hi
    // p: the lane's first byte; all 32 inside the row.  Words that hold none of them are not read.
    __device__ inline void load(const uint8_t* p) {
        if constexpr (ROWS == FP8_ALIGNED) {
            lo = *reinterpret_cast<const u32x4*>(p);
            hi = *reinterpret_cast<const u32x4*>(p + 64);
        } else {
            const uintptr_t u = reinterpret_cast<uintptr_t>(p);
            const void* q = __builtin_assume_aligned(reinterpret_cast<const void*>(u & ~(uintptr_t)3), 4);
            __builtin_memcpy(&lo, q, 16);
            __builtin_memcpy(&hi, static_cast<const char*>(q) + 16, 16);
            next = *reinterpret_cast<const unsigned*>((u + 31) & ~(uintptr_t)3);
        }
    }
    // shift: the row's address modulo 4.
    __device__ inline i32x8 get(unsigned shift) const {
        i32x8 v = __builtin_shufflevector(__builtin_bit_cast(i32x4, lo), __builtin_bit_cast(i32x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (ROWS == FP8_ANY) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = (int)__builtin_amdgcn_alignbyte(i < 7 ? (unsigned)v[i + 1] : next, (unsigned)v[i], shift);
        }
        return v;
    }
};

// 16 codes from byte k of a row of K, zeros past its end.  Nothing past the row is read, and bytes there may be anything,
// NaN codes too: the row's last 16 bytes shifted down (rows shorter than 16: byte by byte).
__device__ inline u32x4 codes_tail(const uint8_t* row, int k, int K) {
    unsigned __int128 u = 0;
    if (K >= 16) {
        const int over = k + 16 - K;
        __builtin_memcpy(&u, row + min(k, K - 16), 16);
        if (over > 0) u = over < 16 ? u >> (8 * over) : 0;
    } else {
        for (int i = K - 1; i >= k; --i) u = u << 8 | row[i];
    }
    return __builtin_bit_cast(u32x4, u);
}
__device__ inline i32x8 join(u32x4 lo, u32x4 hi) {
    return __builtin_shufflevector(__builtin_bit_cast(i32x4, lo), __builtin_bit_cast(i32x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's 32 codes of the last, short block (k: its first).
template <int ROWS> __device__ inline i32x8 lane_tail(const uint8_t* row, int k, int K) {
    return join(codes_tail(row, k, K), codes_tail(row, k + kSecondHalf<ROWS>, K));
}

// Host side: one fp8 product, dense or for the rows of a layer of experts.
struct Fp8Gemm {
    const uint8_t* A; int64_t sa_m;
    const float* a_scale; int64_t sas_m, sas_k;
    const uint8_t* W; int64_t sw_n, sw_g, sw_e;
    const float* w_scale; int64_t sws_n, sws_k, sws_g, sws_e;
    void* C; int64_t sc_m;
    int32_t M, N, K, dtype_c;
    // Experts only (the arrays of expert_plan_kernel).
    const int* row_token;
    const float* row_weight;
    const int4* tiles;
    const int* ntiles;
    const float* route_w;       // routing weights and ids per slot, where there is no plan
    const int* ids;
    int32_t slots;              // per token
    int32_t experts;
    int32_t max_tiles;
    int32_t first_tile;         // of this launch, where the tiles need several
    int32_t first_col;          // of this launch, where the columns need several
    int32_t tokens;             // rows that row_token names
    int32_t tile_rows;          // rows of the plan's tiles
    int32_t exact;              // gate-and-up product in tiles: exact products within a block
    float* mid_scale;           // scales of the quantised inner rows, [I / 128][ld_mid_scale]
    int64_t ld_mid_scale;
    float* row_scale;           // powers of two of the down product's f16 rows, [rows][ld_row_scale], one per 64 columns
    int64_t ld_row_scale;
};

// Rows of K codes as whole 16-byte chunks at 16-byte aligned addresses.
inline bool fast_rows(const void* p, int64_t rows, int64_t stride, int64_t K) {
    return aligned16(p) && K % 16 == 0 && (rows <= 1 || stride % 16 == 0);
}

// Split of a product over k: workgroups per tile, the tiles' arrival counters and partial sums.
struct Fp8Split {
    int parts;
    int* cnt;
    char* slots;
};

// Workspace of a layer of experts per (device, stream).
int experts_workspace(hipStream_t stream, size_t bytes, void** out);

int launch_quantize_fp8(const tv_quantize_fp8_args& a, hipStream_t stream);
int launch_rms_norm_fp8(const tv_rms_norm_fp8_args& a, hipStream_t stream);
int launch_route(const tv_route_args& a, hipStream_t stream);
enum Fp8Mode { FP8_DENSE = 0, FP8_GATE_UP = 1, FP8_DOWN = 2, FP8_SLOT_UP = 3 };
int launch_gemm_fp8(const Fp8Gemm& g, int mode, hipStream_t stream);
// BM x BN tiles through LDS.  TV_E_UNSUPPORTED for operands it does not take (fp8_tile_ok).
bool fp8_tile_ok(const Fp8Gemm& g, int mode);
// Copies of the operands that are not whole 16-byte rows, zero up to the next 16 bytes.  What they need is asked for apart, so that a
// call of several launches can choose other kernels while nothing is launched.
bool fp8_pad_ok(const Fp8Gemm& g, int mode); // no: offsets would stay too large, or the experts' weights have no one stride
struct Fp8PadBytes {
    size_t a, w; // 0: no copy
};
Fp8PadBytes fp8_pad_bytes(const Fp8Gemm& g, int mode);
struct Fp8Pads {
    void *a, *w;
};
int fp8_pad_buffers(const Fp8PadBytes& bytes, hipStream_t stream, Fp8Pads* pads); // TV_E_UNSUPPORTED: no room
int pad_fp8_operands(Fp8Gemm& g, int mode, const Fp8Pads& pads, hipStream_t stream); // g then describes the copies
int launch_gemm_fp8_tile(const Fp8Gemm& g, int mode, hipStream_t stream);
// The second product of a few tokens from inner rows in fp32, summed over their slots.
bool fp8_token_ok(const Fp8Gemm& g, int tokens);
int launch_gemm_fp8_token(const Fp8Gemm& g, const float* mid, int64_t ld, int tokens, hipStream_t stream);
// 16 to 64 rows and 128 columns a workgroup, W straight from memory.
int launch_gemm_fp8_wide(const Fp8Gemm& g, int mode, hipStream_t stream);
int launch_experts_fp8(const tv_experts_fp8_args& a, hipStream_t stream);

} // namespace tvk
