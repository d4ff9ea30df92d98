// Products of e4m3 operands with a scale per block of 128 along k:
//     C[m, n] = sum_b as[m, b] * ws[n / 128, b] * sum_{k in b} A[m, k] * W[n, k].
// One v_mfma_f32_16x16x128_f8f6f4 is one block's inner sum of 16 x 16 outputs, so the block's scale is one
// multiply-add per output on the vector ALUs: acc += (as * ws) * mfma(w, a, 0).  W is the instruction's
// first operand and A its second, so that a lane holds four consecutive columns n = 4 (lane / 16) + q of one
// row m = lane % 16: the scale is one value per lane, and the four outputs are one store.
// (The order of k inside a fragment is the same for both operands, so any assignment of the 128 k of a block to
// lanes and registers gives the same sums.)
#include "fp8_common.h"

namespace tvk {

// Products of few rows: the weights stream from memory, so a workgroup takes 16 columns and 16 MT rows, and
// its KW waves take every KW-th block of k; their sums meet in LDS.  Operands go straight from memory to
// registers (no wave shares W with another, and A's few rows come from the caches).  Bound by W's bytes: [1,4096]x[11008,4096]
// 9.7 us, 4.7 TB/s; up-projections of one token through 8 experts of 1376 (90 MB) 16.6 us, 5.4 TB/s.
//  FP8_DENSE    C [M, N] in dtype_c;
//  FP8_GATE_UP  rows of one expert, gathered through row_token; both halves of W1, C = silu(gate) * up in fp32;
//  FP8_SLOT_UP  the same without a plan: a tile is one slot;
//  FP8_DOWN     rows of one expert in the plan's order, times their routing weight, in fp32.
//  EXACT: exact products of a block (mfma_fp8_exact), for fp32 results, and for the inner rows, which are rounded to e4m3 next: an error
//  of 1.5e-5 moves one value in two thousand to the other code beside it, which shows where the rows are few.  (W's bytes
//  bound the call either way.)
template <typename TC, int MODE, bool EXACT, int MT, int KW, int U, int ROWS>
__global__ __launch_bounds__(64 * KW) void gemm_fp8_direct_kernel(Fp8Gemm g) {
    constexpr int NG = MODE == FP8_GATE_UP || MODE == FP8_SLOT_UP ? 2 : 1;
    constexpr int PITCH = 17; // floats per row of 16 sums
    __shared__ float sums[KW][NG][MT * 16 * PITCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, grp = lane >> 4;
    const int n0 = g.first_col + (int)blockIdx.x * 16;
    int m0, m1, expert = 0; // rows of this tile
    if constexpr (MODE == FP8_DENSE) {
        m0 = (g.first_tile + (int)blockIdx.y) * MT * 16;
        m1 = min(g.M, m0 + MT * 16);
    } else if constexpr (MODE == FP8_SLOT_UP) {
        m0 = g.first_tile + (int)blockIdx.y; // a slot is its own row and tile
        m1 = m0 + 1;
        expert = g.ids[m0];
        if ((unsigned)expert >= (unsigned)g.experts) return;
    } else {
        const int tile = g.first_tile + (int)blockIdx.y;
        if (tile >= *g.ntiles) return;
        const int4 at = g.tiles[tile];
        expert = at.x;
        m0 = at.y;
        m1 = at.z;
    }
    const uint8_t* a_row[MT];
    const float* a_scale[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = min(m0 + 16 * i + r, m1 - 1); // rows past the tile repeat its last one; they are not stored
        const int64_t row = MODE == FP8_GATE_UP ? g.row_token[m] : MODE == FP8_SLOT_UP ? m / g.slots : m;
        a_row[i] = g.A + row * g.sa_m;
        a_scale[i] = g.a_scale + row * g.sas_m;
    }
    const int n = min(n0 + r, g.N - 1);
    const uint8_t* w_row = g.W + (int64_t)expert * g.sw_e + (int64_t)n * g.sw_n;
    const float* w_scale = g.w_scale + (int64_t)expert * g.sws_e + (int64_t)(n0 / TV_FP8_BLOCK) * g.sws_n;
    f32x4 acc[NG][MT];
#pragma unroll
    for (int h = 0; h < NG; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[h][i] = f32x4{0, 0, 0, 0};
    const int kb = (g.K + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK;
    const int whole = g.K / TV_FP8_BLOCK, lane_k = grp * kLaneStep<ROWS>;
    unsigned w_shift[NG], a_shift[MT];
#pragma unroll
    for (int h = 0; h < NG; ++h) w_shift[h] = (unsigned)reinterpret_cast<uintptr_t>(w_row + h * g.sw_g) & 3;
#pragma unroll
    for (int i = 0; i < MT; ++i) a_shift[i] = (unsigned)reinterpret_cast<uintptr_t>(a_row[i]) & 3;
    // used: uniform; a select, not a branch, so that the loads stay ahead of it (and a NaN that is not used does not count).
    auto multiply = [&](const i32x8& w, const i32x8& x, float s, f32x4& sum, bool used) {
        f32x4 t;
        if constexpr (EXACT) t = mfma_fp8_exact(w, x);
        else t = mfma_fp8(w, x);
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] = used ? __builtin_fmaf(s, t[q], sum[q]) : sum[q];
    };
    // The last, short block belongs to the wave whose turn it is; it is loaded first and used last.
    const bool tail = whole < kb && wave == whole % KW;
    i32x8 wt[NG], at[MT];
    float wst[NG], ast[MT];
    if (tail) {
        const int k = whole * TV_FP8_BLOCK + lane_k;
#pragma unroll
        for (int h = 0; h < NG; ++h) {
            wt[h] = lane_tail<ROWS>(w_row + h * g.sw_g, k, g.K);
            wst[h] = w_scale[h * g.sws_g + (int64_t)whole * g.sws_k];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            at[i] = lane_tail<ROWS>(a_row[i], k, g.K);
            ast[i] = a_scale[i][(int64_t)whole * g.sas_k];
        }
    }
    // U whole blocks at a time, all loads before the first product, so that a wave's share of a short k is in flight at
    // once.  The loads have no condition (a branch around them would keep them from going out together): blocks past the
    // end read the last one again and are not used.
    for (int b0 = wave; b0 < whole; b0 += KW * U) {
        LaneCodes<ROWS> wf[U][NG], af[U][MT];
        float ws[U][NG], as[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = min(b0 + u * KW, whole - 1), k = b * TV_FP8_BLOCK + lane_k;
#pragma unroll
            for (int h = 0; h < NG; ++h) {
                wf[u][h].load(w_row + h * g.sw_g + k);
                ws[u][h] = w_scale[h * g.sws_g + (int64_t)b * g.sws_k];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                af[u][i].load(a_row[i] + k);
                as[u][i] = a_scale[i][(int64_t)b * g.sas_k];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < NG; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    multiply(wf[u][h].get(w_shift[h]), af[u][i].get(a_shift[i]), as[u][i] * ws[u][h], acc[h][i], b0 + u * KW < whole);
        }
    }
    if (tail) {
#pragma unroll
        for (int h = 0; h < NG; ++h)
#pragma unroll
            for (int i = 0; i < MT; ++i) multiply(wt[h], at[i], ast[i] * wst[h], acc[h][i], true);
    }
#pragma unroll
    for (int h = 0; h < NG; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) sums[wave][h][(16 * i + r) * PITCH + 4 * grp + q] = acc[h][i][q];
    __syncthreads();
    for (int o = threadIdx.x; o < MT * 256; o += 64 * KW) {
        const int m = m0 + (o >> 4), c = n0 + (o & 15);
        if (m >= m1 || c >= g.N) continue;
        float v[NG];
#pragma unroll
        for (int h = 0; h < NG; ++h) {
            v[h] = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; ++w) v[h] += sums[w][h][(o >> 4) * PITCH + (o & 15)];
        }
        float out = v[0];
        if constexpr (NG == 2) out = act_logistic(v[0], act_coef(TV_ACT_SILU)) * v[NG - 1];
        if constexpr (MODE == FP8_DOWN) out *= g.row_weight[m];
        static_cast<TC*>(g.C)[(int64_t)m * g.sc_m + c] = (TC)out;
    }
}

// The second product of a few tokens, one workgroup of 16 waves for 16 columns of one token: the blocks of all the
// token's slots, one after the other, are a single long k, so the sum over slots is the accumulation (the routing
// weight is part of the block's scale) and C is written once.  The inner rows [slots][ld] come in fp32: they are a
// few kilobytes, which every workgroup quantises into LDS itself while its first weights are on their way.  With
// plan, quantisation, product and sum as launches of their own one token of 64 experts of 1376, k = 8, took 46 us; it takes 31 to 33
// (this kernel 12 for 45 MB: its first loads and the quantisation are a third of it; four or six blocks in flight took 32.5 and 33.2 where
// three took 31).
constexpr int kTokenWaves = 16, kTokenU = 3;

template <typename TC, int ROWS>
__global__ __launch_bounds__(64 * kTokenWaves) void gemm_fp8_token_kernel(Fp8Gemm g, const float* mid, int64_t ld) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, grp = lane >> 4;
    const int n0 = blockIdx.x * 16, kb = (g.K + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK, total = g.slots * kb;
    const int* ids = g.ids + (int64_t)blockIdx.y * g.slots;
    const float* weights = g.route_w + (int64_t)blockIdx.y * g.slots;
    mid += (int64_t)blockIdx.y * g.slots * ld;
    char* codes = lds;                                                  // [total] blocks of 128
    float* scales = reinterpret_cast<float*>(lds + total * TV_FP8_BLOCK); // [total]
    const int n = min(n0 + r, g.N - 1);

    // Block q of the token: block q % kb of slot q / kb.
    struct Block {
        LaneCodes<ROWS> f;
        unsigned shift;
        float s;
        bool used;
    } w[kTokenU];
    auto load = [&](Block& b, int q) {
        const int qc = min(q, total - 1), slot = qc / kb, k = (qc - slot * kb) * TV_FP8_BLOCK + grp * kLaneStep<ROWS>;
        const int e = ids[slot];
        b.used = q < total && (unsigned)e < (unsigned)g.experts;
        const int ec = b.used ? e : 0;
        const uint8_t* row = g.W + (int64_t)ec * g.sw_e + (int64_t)n * g.sw_n;
        if constexpr (ROWS == FP8_ALIGNED) {
            // Chunks past K read the row's last one and count as zeros.
            b.f.lo = *reinterpret_cast<const u32x4*>(row + min(k, g.K - 16));
            b.f.hi = *reinterpret_cast<const u32x4*>(row + min(k + 64, g.K - 16));
            if (k >= g.K) b.f.lo = u32x4{0, 0, 0, 0};
            if (k + 64 >= g.K) b.f.hi = u32x4{0, 0, 0, 0};
        } else if ((qc - slot * kb + 1) * TV_FP8_BLOCK <= g.K) { // uniform
            b.f.load(row + k);
            b.shift = (unsigned)reinterpret_cast<uintptr_t>(row) & 3;
        } else {
            b.f.lo = codes_tail(row, k, g.K);
            b.f.hi = codes_tail(row, k + kSecondHalf<ROWS>, g.K);
            b.shift = 0;
        }
        b.s = g.w_scale[(int64_t)ec * g.sws_e + (int64_t)(n0 / TV_FP8_BLOCK) * g.sws_n + (int64_t)(qc - slot * kb) * g.sws_k] * weights[slot];
    };
#pragma unroll
    for (int u = 0; u < kTokenU; ++u) load(w[u], wave + u * kTokenWaves);
    // Quantise: 16 lanes a block, as quantize_rows_kernel.  Slots without expert have no row.
    for (int q = threadIdx.x >> 4; q < total; q += 4 * kTokenWaves) {
        const int slot = q / kb, k = (q - slot * kb) * TV_FP8_BLOCK + r * 8;
        float v[8];
        Eight<float> x;
        x.load(mid + slot * ld, k, ld); // rows are padded to whole blocks
        const bool has = (unsigned)ids[slot] < (unsigned)g.experts;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = has && k + j < g.K ? x.e[j] : 0.0f;
        unsigned mx = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = umax(mx, abs_bits(v[j]));
        const Fp8Block f = fp8_block(row16_max(mx));
        store_codes8(reinterpret_cast<uint8_t*>(codes) + q * TV_FP8_BLOCK + r * 8, 8, v, f);
        if (r == 0) scales[q] = f.scale;
    }
    __syncthreads();
    f32x4 acc = {0, 0, 0, 0};
    for (int q0 = wave; q0 < total; q0 += kTokenWaves * kTokenU) {
#pragma unroll
        for (int u = 0; u < kTokenU; ++u) {
            const int q = q0 + u * kTokenWaves, qc = min(q, total - 1);
            const char* x = codes + qc * TV_FP8_BLOCK + grp * kLaneStep<ROWS>;
            const i32x8 wq = w[u].f.get(w[u].shift), xq = join(*reinterpret_cast<const u32x4*>(x), *reinterpret_cast<const u32x4*>(x + kSecondHalf<ROWS>));
            f32x4 t;
            if constexpr (__is_same(TC, float)) t = mfma_fp8_exact(wq, xq);
            else t = mfma_fp8(wq, xq);
            const float s = scales[qc] * w[u].s;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = w[u].used ? __builtin_fmaf(s, t[i], acc[i]) : acc[i];
            load(w[u], q + kTokenWaves * kTokenU);
        }
    }
    __syncthreads(); // the codes are done with
    float* sums = reinterpret_cast<float*>(lds); // [waves][16]
    if (r == 0) *reinterpret_cast<f32x4*>(sums + wave * 16 + 4 * grp) = acc;
    __syncthreads();
    if (threadIdx.x < 16 && n0 + (int)threadIdx.x < g.N) {
        float out = 0.0f;
#pragma unroll
        for (int i = 0; i < kTokenWaves; ++i) out += sums[i * 16 + threadIdx.x];
        static_cast<TC*>(g.C)[(int64_t)blockIdx.y * g.sc_m + n0 + threadIdx.x] = (TC)out;
    }
}

// LDS of one token: its slots' codes and scales (and at least the waves' sums).
static size_t token_lds(const Fp8Gemm& g) {
    const size_t blocks = (size_t)g.slots * ((g.K + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK), bytes = blocks * (TV_FP8_BLOCK + 4);
    return bytes > kTokenWaves * 64 ? bytes : kTokenWaves * 64;
}

// tokens: rows of the grid, whose threads are limited to 2^32.
bool fp8_token_ok(const Fp8Gemm& g, int tokens) {
    return token_lds(g) <= 64 * 1024 && ((int64_t)g.N + 15) / 16 * tokens < ((int64_t)1 << 32) / (64 * kTokenWaves);
}

int launch_gemm_fp8_token(const Fp8Gemm& g, const float* mid, int64_t ld, int tokens, hipStream_t stream) {
    const dim3 grid(((int64_t)g.N + 15) / 16, tokens);
    auto run = [&](auto zero) {
        if (fast_rows(g.W, g.N, g.sw_n, g.K) && g.sw_e % 16 == 0)
            hipLaunchKernelGGL((gemm_fp8_token_kernel<decltype(zero), FP8_ALIGNED>), grid, dim3(64 * kTokenWaves), token_lds(g), stream, g, mid, ld);
        else
            hipLaunchKernelGGL((gemm_fp8_token_kernel<decltype(zero), FP8_ANY>), grid, dim3(64 * kTokenWaves), token_lds(g), stream, g, mid, ld);
        return (int)hipGetLastError();
    };
    switch (g.dtype_c) {
        case TV_BFLOAT16: return run((__bf16)0.0f);
        case TV_FLOAT16: return run((_Float16)0.0f);
        default: return run(0.0f);
    }
}

template <typename TC, int MODE, bool EXACT, int MT, int KW, int U> static int direct(const Fp8Gemm& g, bool fast, hipStream_t stream) {
    const int64_t mt = MODE == FP8_DENSE ? ((int64_t)g.M + 16 * MT - 1) / (16 * MT) : MODE == FP8_SLOT_UP ? g.M : g.max_tiles;
    const int64_t nt = ((int64_t)g.N + 15) / 16;
    // The grid's rows are limited to 65535, its threads to 2^32.
    const int64_t room = ((int64_t)1 << 32) / (64 * KW) - 1, cols = nt < room ? nt : room, rows = room / cols < 32768 ? room / cols : 32768;
    for (int64_t x = 0; x < nt; x += cols)
        for (int64_t y = 0; y < mt; y += rows) {
            Fp8Gemm p = g;
            p.first_col = (int32_t)(x * 16);
            p.first_tile = (int32_t)y;
            const dim3 grid((unsigned)(nt - x < cols ? nt - x : cols), (unsigned)(mt - y < rows ? mt - y : rows));
            if (fast) hipLaunchKernelGGL((gemm_fp8_direct_kernel<TC, MODE, EXACT, MT, KW, U, FP8_ALIGNED>), grid, dim3(64 * KW), 0, stream, p);
            else hipLaunchKernelGGL((gemm_fp8_direct_kernel<TC, MODE, EXACT, MT, KW, U, FP8_ANY>), grid, dim3(64 * KW), 0, stream, p);
            const int rc = hipGetLastError();
            if (rc) return rc;
        }
    return 0;
}

// One block of k in flight per wave up to 16 blocks, four beyond.  us in bf16, one row, one block in flight / four:
// [1024 -> 4096] 2.8 / 4.5, [2048 -> 11008] 6.3 / 9.4, [4096 -> 4096] 5.5 / 5.4, [4096 -> 11008] 10.4 / 9.9.
template <typename TC, int MODE, bool EXACT> static int direct_u(const Fp8Gemm& g, bool fast, hipStream_t stream) {
    if (g.K <= 16 * TV_FP8_BLOCK) return direct<TC, MODE, EXACT, 1, 8, 1>(g, fast, stream);
    return direct<TC, MODE, EXACT, 1, 8, 4>(g, fast, stream);
}

// rows: of a workgroup.
template <typename TC> static int dense(const Fp8Gemm& g, bool fast, int rows, hipStream_t stream) {
    constexpr bool exact = __is_same(TC, float);
    if (rows == 16) return direct_u<TC, FP8_DENSE, exact>(g, fast, stream);
    if (rows == 32) return direct<TC, FP8_DENSE, exact, 2, 8, 1>(g, fast, stream);
    return direct<TC, FP8_DENSE, exact, 4, 8, 1>(g, fast, stream);
}

// What a dense product of more than 16 rows takes on each kernel, in us, and the kernel that takes least.  Fitted to bf16
// products of 17 to 4096 rows, K 512 to 11008, N 512 to 11008; a few of them, predicted / measured:
//                             direct       wide        128x128 tiles  256x256 tiles
//   [32,1024]x[1024,1024]     3.3 / 3.4    8.1 / 7.8    10 / 9.0       18 / 14.5
//   [32,4096]x[11008,4096]     18 / 19      17 / 16.5   19 / 22        60 / 43
//   [128,11008]x[4096,11008]   61 / 55       -          25 / 24       155 / 107
//   [256,2048]x[4096,2048]     25 / 24       -          15 / 15        32 / 25
//   [1024,4096]x[11008,4096]  470 / -        -          75 / 61        60 / 55
// Over 92 products of 17 to 1024 rows, 500 to 11008 k and 300 to 11008 columns, in bf16 and fp32, odd sizes among them, the kernel
// chosen takes 1.04 of the fastest one's time (geometric mean; 1.27 at most).
//  * direct: a workgroup per 16, 32 or 64 rows and 16 columns: where they do not fill the CUs a workgroup's own latency, which is
//    less the fewer its rows, else their time on a CU, which is less a row the more its rows.  us in bf16, workgroups of 16 / 32 /
//    64 rows: [64,1024]x[1024,1024] 3.2 / 3.7 / 5.0, [64,2048]x[2048,2048] 5.8 / 5.1 / 7.5, [100,1024]x[4096,1024] 8.4 / 7.7 /
//    7.3.  With exact sums those of 64 rows take a quarter more ([333,1024]x[4096,1024] 24 us, bf16 20);
//  * wide: the latency of a part's blocks, the parts' sums, W's bytes;
//  * tiles: rounds of the CUs' workgroups over k-tiles (2 of 128x128, 1 of 256x256 on a CU), the parts' sums through memory,
//    and the padded copies of operands that need them.  fp32 results run on the bf16 instructions, at 1.7 times the k-tile.
struct Fp8Price {
    double direct, wide, tile128, tile256;
    int direct_rows; // of a direct workgroup
};
static Fp8Price price(const Fp8Gemm& g, bool fast) {
    const double M = g.M, N = g.N, K = g.K, kt = (double)((g.K + 127) / 128), cus = device_cus();
    const auto up = [](double x, double y) { return (double)(int64_t)((x + y - 1) / y); };
    const double shifted = fast ? 1.0 : 1.25, exact = g.dtype_c == TV_FLOAT32 ? 1.7 : 1.0;
    Fp8Price p;
    p.direct = 1e30;
    const double m64 = M < 64 ? M : 64;
    const struct { int rows; double start, alone, full; } kinds[3] = {
        {16, 2.4, 0.85, 0.87}, {32, 2.4, 1.1, 1.42}, {64, 3.0, 0.9 + 0.022 * m64, (1.5 + 0.018 * m64) * (exact > 1 ? 1.25 : 1)}};
    for (const auto& d : kinds) {
        const double full = up(M, d.rows) * up(N, 16) / cus * d.full, us = d.start + shifted * K / 1000 * (d.alone > full ? d.alone : full);
        if (us < p.direct) {
            p.direct = us;
            p.direct_rows = d.rows;
        }
    }
    const auto parts_of = [](double room, double most, double limit) {
        double x = room < most ? room : most;
        x = x < limit ? x : limit;
        return x < 1 ? 1.0 : (double)(int64_t)x;
    };
    const double wt = up(N, 128), wp = parts_of(2 * cus / wt, kt / 4, 16);
    const double wr = M > 32 ? 64 : 32;
    p.wide = M > 64 ? 1e30 : 4.0 + shifted * (up(kt, wp) * (0.55 + 0.01 * wr) + N * K / 1.2e7) + (wp > 1 ? wp * (0.25 + wr * N * 1.2e-6) : 0);
    const double pad = fp8_tile_ok(g, FP8_DENSE) ? 0 : 2.5 + 2 * (M + N) * K / 4.5e6;
    const double t1 = up(M, 128) * up(N, 128), p1 = parts_of(2 * cus / t1, kt / 4, 8), w1 = t1 * p1;
    p.tile128 = 5.0 + pad + up(w1, 2 * cus) * up(kt, p1) * exact * (w1 <= cus ? 0.75 : 1.1) + (p1 > 1 ? p1 * (1 + M * N * 8 / 1e7) : 0);
    const double t2 = up(M, 256) * up(N, 256);
    p.tile256 = exact > 1 ? 1e30 : 4.0 + pad + up(t2, cus) * kt * 1.75;
    return p;
}

int launch_gemm_fp8(const Fp8Gemm& g, int mode, hipStream_t stream) {
    const bool fast = fast_rows(g.A, g.M, g.sa_m, g.K) && fast_rows(g.W, g.N, g.sw_n, g.K) && g.sw_e % 16 == 0 && g.sw_g % 16 == 0;
    if (mode == FP8_GATE_UP) return direct_u<float, FP8_GATE_UP, true>(g, fast, stream);
    if (mode == FP8_SLOT_UP) return direct_u<float, FP8_SLOT_UP, true>(g, fast, stream);
    if (mode == FP8_DOWN) return g.dtype_c == TV_FLOAT32 ? direct_u<float, FP8_DOWN, true>(g, fast, stream) : direct_u<float, FP8_DOWN, false>(g, fast, stream);
    int rows = 16;
    if (g.M > 16 && g.K > 0) {
        const Fp8Price p = price(g, fast);
        rows = p.direct_rows;
        const double tile = p.tile128 < p.tile256 ? p.tile128 : p.tile256;
        if (tile < p.direct && tile < p.wide) {
            Fp8Gemm t = g;
            t.tile_rows = p.tile128 < p.tile256 ? 128 : 256;
            int rc = 0;
            if (!fp8_tile_ok(t, mode)) {
                Fp8Pads pads;
                rc = fp8_pad_ok(t, mode) ? fp8_pad_buffers(fp8_pad_bytes(t, mode), stream, &pads) : (int)TV_E_UNSUPPORTED;
                if (rc == 0) rc = pad_fp8_operands(t, mode, pads, stream);
            }
            if (rc == 0) rc = launch_gemm_fp8_tile(t, mode, stream);
            if (rc != TV_E_UNSUPPORTED) return rc;
        }
        if (p.wide < p.direct) {
            const int rc = launch_gemm_fp8_wide(g, mode, stream);
            if (rc != TV_E_UNSUPPORTED) return rc;
        }
    }
    switch (g.dtype_c) {
        case TV_BFLOAT16: return dense<__bf16>(g, fast, rows, stream);
        case TV_FLOAT16: return dense<_Float16>(g, fast, rows, stream);
        default: return dense<float>(g, fast, rows, stream);
    }
}

} // namespace tvk
