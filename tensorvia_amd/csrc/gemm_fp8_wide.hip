// Products of 17 to 64 rows, and of an expert's few rows: 16 MT rows and 128 columns a workgroup of 8 waves, 16
// columns a wave (of gate and of up).
//
// The weights stream from memory and bound the call, so they go straight from memory to registers, in the order the
// matrix instruction takes them, a chunk of KC blocks ahead of their use.  The rows are the same for all 8 waves: a chunk
// of them goes through LDS once per workgroup (read by each wave from its own column of 16 workgroups' worth of L2
// traffic, they made 64 rows cost three times one).  With 128 columns a workgroup holds a whole block of the inner
// rows' codes, so the gate-and-up product quantises them in its epilogue.
// 64 tokens of 64 experts of 1376, k = 8: gate and up 138 us, 5.2 TB/s, down 78 us, 4.6 TB/s, bound by W's bytes.
// Few tiles: the workgroups split k, and the last to arrive sums the parts in order (100 tokens of 8 experts of 1376, k = 2, 88 tiles
// for the gate-and-up product: 62 us whole, 50 in parts).
#include "fp8_common.h"

#include <type_traits>

namespace tvk {

template <int MODE_, typename TC_, bool EXACT_, int MT_, int ROWS_> struct Fp8Wide {
    using TC = TC_;
    static constexpr int MODE = MODE_, MT = MT_, BM = 16 * MT_, NG = MODE_ == FP8_GATE_UP ? 2 : 1;
    static constexpr int ROWS = ROWS_;
    static constexpr bool EXACT = EXACT_; // exact products of a block, as the direct kernel's
    static constexpr int WAVES = 8, THREADS = 512;
    static constexpr int KC = 2;                         // blocks of k per chunk
    static constexpr int PITCH = KC * 128 + 16;          // bytes of a row's chunk in LDS: 16 rows on distinct banks
    static constexpr int CHUNKS = BM * KC * 8;           // 16-byte pieces of a chunk of rows
    static constexpr int PER = (CHUNKS + THREADS - 1) / THREADS;
    // Two workgroups a CU: 128 registers a wave, which the gate-and-up product of more than 16 rows, or of shifted rows, does not fit.
    static constexpr int WGS = NG == 2 && (MT > 1 || ROWS == FP8_ANY) ? 1 : 2;
};

template <class C>
__global__ __launch_bounds__(512, 2 * C::WGS) void gemm_fp8_wide_kernel(Fp8Gemm g, int tiles_n, Fp8Split sp) {
    constexpr int MT = C::MT, NG = C::NG, KC = C::KC, MODE = C::MODE;
    __shared__ __attribute__((aligned(16))) char rows[2][C::BM * C::PITCH];
    __shared__ float scales[2][KC][C::BM];
    __shared__ unsigned part[C::BM][C::WAVES];
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, grp = lane >> 4;

    int id = blockIdx.x;
    if constexpr (MODE != FP8_DENSE) {
        const int total = *g.ntiles * tiles_n * sp.parts, per = (total + 7) >> 3; // contiguous runs of tiles per XCD
        id = (id >> 3) < per ? (id & 7) * per + (id >> 3) : total;
        if (id >= total) return;
    }
    const int s = id % sp.parts; // a tile's parts side by side
    id /= sp.parts;
    int m0, m1, n0, expert = 0;
    if constexpr (MODE == FP8_DENSE) {
        const int tm = id / tiles_n;
        m0 = tm * C::BM;
        m1 = min(g.M, m0 + C::BM);
        n0 = (id - tm * tiles_n) * 128;
    } else {
        const int tile = id / tiles_n;
        const int4 at = g.tiles[tile];
        expert = at.x;
        m0 = at.y;
        m1 = at.z;
        n0 = (id - tile * tiles_n) * 128;
    }
    const int kb = (g.K + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK;
    const int b_lo = (int)((int64_t)kb * s / sp.parts), b_end = (int)((int64_t)kb * (s + 1) / sp.parts);
    const int whole = g.K / 128, b_hi = min(b_end, whole); // whole blocks; a last, short one apart
    const int nc = b_hi > b_lo ? (b_hi - b_lo + KC - 1) / KC : 0;

    // Rows: piece p of a chunk is 16 bytes c of row m.
    const uint8_t* a_ptr[C::PER];
    int a_k[C::PER];
    unsigned a_lds[C::PER];
#pragma unroll
    for (int j = 0; j < C::PER; ++j) {
        const int p = min(tid + j * C::THREADS, C::CHUNKS - 1), m = p / (KC * 8), c = p % (KC * 8);
        const int row = min(m0 + m, m1 - 1); // rows past the tile repeat its last one; they are not stored
        a_ptr[j] = g.A + (MODE == FP8_GATE_UP ? (int64_t)g.row_token[row] : (int64_t)row) * g.sa_m;
        a_k[j] = c * 16;
        a_lds[j] = m * C::PITCH + c * 16;
    }
    // Scales of a chunk: thread t's is row t % BM, block t / BM.
    constexpr int NS = C::BM * KC;
    const int sm = min(m0 + tid % C::BM, m1 - 1);
    const float* as_ptr = g.a_scale + (MODE == FP8_GATE_UP ? (int64_t)g.row_token[sm] : (int64_t)sm) * g.sas_m;
    u32x4 a_reg[C::PER];
    unsigned a_next[C::PER];
    float as_reg = 0.0f;
    // Pieces of rows that are not aligned: the words that hold them, as LaneCodes.  Pieces past the whole blocks read the
    // row's last whole block again and are not used.
    auto load_rows = [&](int c) {
        const int b0 = b_lo + c * KC;
#pragma unroll
        for (int j = 0; j < C::PER; ++j) {
            const uint8_t* p = a_ptr[j] + min(b0 * 128 + a_k[j], whole * 128 - 16);
            if constexpr (C::ROWS == FP8_ALIGNED) {
                a_reg[j] = *reinterpret_cast<const u32x4*>(p);
            } else {
                const uintptr_t u = reinterpret_cast<uintptr_t>(p);
                __builtin_memcpy(&a_reg[j], __builtin_assume_aligned(reinterpret_cast<const void*>(u & ~(uintptr_t)3), 4), 16);
                a_next[j] = *reinterpret_cast<const unsigned*>((u + 15) & ~(uintptr_t)3);
            }
        }
        if (tid < NS) as_reg = as_ptr[(int64_t)min(b0 + tid / C::BM, kb - 1) * g.sas_k];
    };
    auto store_rows = [&](int c) {
#pragma unroll
        for (int j = 0; j < C::PER; ++j) {
            u32x4 v = a_reg[j];
            if constexpr (C::ROWS == FP8_ANY) {
                const unsigned sh = (unsigned)reinterpret_cast<uintptr_t>(a_ptr[j]) & 3;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? a_reg[j][i + 1] : a_next[j], a_reg[j][i], sh);
            }
            if (C::CHUNKS % C::THREADS == 0 || tid + j * C::THREADS < C::CHUNKS) *reinterpret_cast<u32x4*>(rows[c & 1] + a_lds[j]) = v;
        }
        if (tid < NS) scales[c & 1][tid / C::BM][tid % C::BM] = as_reg;
    };

    // Weights: lane's row of the wave's 16 columns.
    const int n = min(n0 + wave * 16 + r, g.N - 1), lane_k = grp * kLaneStep<C::ROWS>;
    const uint8_t* w_row = g.W + (int64_t)expert * g.sw_e + (int64_t)n * g.sw_n;
    const float* w_scale = g.w_scale + (int64_t)expert * g.sws_e + (int64_t)(n0 / 128) * g.sws_n;
    unsigned w_shift[NG];
#pragma unroll
    for (int h = 0; h < NG; ++h) w_shift[h] = (unsigned)reinterpret_cast<uintptr_t>(w_row + h * g.sw_g) & 3;
    struct Weights {
        LaneCodes<C::ROWS> f[KC][NG];
        float s[KC][NG];
    };
    auto load_w = [&](Weights& w, int c) {
#pragma unroll
        for (int u = 0; u < KC; ++u) {
            const int b = min(b_lo + c * KC + u, b_hi - 1);
#pragma unroll
            for (int h = 0; h < NG; ++h) {
                w.f[u][h].load(w_row + h * g.sw_g + b * 128 + lane_k);
                w.s[u][h] = w_scale[h * g.sws_g + (int64_t)b * g.sws_k];
            }
        }
    };
    f32x4 acc[NG][MT];
#pragma unroll
    for (int h = 0; h < NG; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[h][i] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const i32x8& w, const i32x8& x, float f, f32x4& sum) {
        if constexpr (C::EXACT) sum += f * mfma_fp8_exact(w, x);
        else sum += f * mfma_fp8(w, x);
    };
    auto compute = [&](Weights& w, int c) {
        const char* base = rows[c & 1] + r * C::PITCH + lane_k;
#pragma unroll
        for (int u = 0; u < KC; ++u) {
            const int b = b_lo + c * KC + u;
            if (b >= b_hi) break; // uniform
            i32x8 y[NG];
#pragma unroll
            for (int h = 0; h < NG; ++h) y[h] = w.f[u][h].get(w_shift[h]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const char* p = base + i * 16 * C::PITCH + u * 128;
                const i32x8 x = join(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + kSecondHalf<C::ROWS>));
                const float as = scales[c & 1][u][16 * i + r];
                if constexpr (C::EXACT) {
                    // A quarter of the codes at a time: few registers.
                    f32x4 t[NG];
#pragma unroll
                    for (int h = 0; h < NG; ++h) t[h] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const bf16x8 xq = exact_codes(x, q);
#pragma unroll
                        for (int h = 0; h < NG; ++h) t[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(exact_codes(y[h], q), xq, t[h], 0, 0, 0);
                    }
#pragma unroll
                    for (int h = 0; h < NG; ++h) acc[h][i] += as * w.s[u][h] * t[h];
                } else {
#pragma unroll
                    for (int h = 0; h < NG; ++h) multiply(y[h], x, as * w.s[u][h], acc[h][i]);
                }
            }
        }
    };

    // A chunk of weights is in flight while the one before is used; rows go to the other half of LDS behind it.
    Weights w0, w1;
    if (nc > 0) {
        load_rows(0);
        load_w(w0, 0);
    }
    if (b_end > b_hi) {
        // The last, short block, straight from memory, while the first chunk is on its way.
        const int k = whole * 128 + lane_k;
        i32x8 y[NG];
        float ws[NG];
#pragma unroll
        for (int h = 0; h < NG; ++h) {
            y[h] = lane_tail<C::ROWS>(w_row + h * g.sw_g, k, g.K);
            ws[h] = w_scale[h * g.sws_g + (int64_t)whole * g.sws_k];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = min(m0 + 16 * i + r, m1 - 1);
            const int64_t row = MODE == FP8_GATE_UP ? (int64_t)g.row_token[m] : (int64_t)m;
            const i32x8 x = lane_tail<C::ROWS>(g.A + row * g.sa_m, k, g.K);
            const float as = g.a_scale[row * g.sas_m + (int64_t)whole * g.sas_k];
#pragma unroll
            for (int h = 0; h < NG; ++h) multiply(y[h], x, as * ws[h], acc[h][i]);
        }
    }
    if (nc > 0) store_rows(0);
    if (nc > 1) load_rows(1);
    __syncthreads();
    for (int c = 0; c < nc; c += 2) {
        if (c + 1 < nc) load_w(w1, c + 1);
        compute(w0, c);
        if (c + 1 < nc) {
            store_rows(c + 1);
            if (c + 2 < nc) {
                load_rows(c + 2);
                load_w(w0, c + 2);
            }
            __syncthreads();
            compute(w1, c + 1);
            if (c + 2 < nc) {
                store_rows(c + 2);
                if (c + 3 < nc) load_rows(c + 3);
            }
        }
        __syncthreads();
    }

    if (sp.parts > 1) {
        // Partial sums in register order, a slot per part; the last part to arrive sums them in part order.
        constexpr int BYTES = C::THREADS * NG * MT * 16;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(sp.slots + (int64_t)id * sp.parts * BYTES, (int64_t)sp.parts * BYTES);
#pragma unroll
        for (int h = 0; h < NG; ++h)
#pragma unroll
            for (int i = 0; i < MT; ++i) slot_store16(rs, s * BYTES + ((h * MT + i) * C::THREADS + tid) * 16, acc[h][i]);
        publish_and_count(sp.cnt + id, sp.parts, &last);
        if (!last) return;
#pragma unroll
        for (int h = 0; h < NG; ++h)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[h][i] = f32x4{0, 0, 0, 0};
        for (int q = 0; q < sp.parts; ++q)
#pragma unroll
            for (int h = 0; h < NG; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[h][i] += slot_load16<f32x4>(rs, q * BYTES + ((h * MT + i) * C::THREADS + tid) * 16);
        slot_count_reset(sp.cnt + id);
    }

    if constexpr (MODE == FP8_GATE_UP) {
        const ActCoef silu = act_coef(TV_ACT_SILU);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            unsigned mx = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bool in = n0 + wave * 16 + 4 * grp + q < g.N; // columns past the end repeat the last one
                acc[0][i][q] = in ? act_logistic(acc[0][i][q], silu) * acc[NG - 1][i][q] : 0.0f;
                mx = umax(mx, abs_bits(acc[0][i][q]));
            }
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 16));
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 32));
            if (grp == 0) part[16 * i + r][wave] = mx;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            unsigned mx = 0;
#pragma unroll
            for (int v = 0; v < C::WAVES; ++v) mx = umax(mx, part[16 * i + r][v]);
            const Fp8Block f = fp8_block(mx);
            const int m = m0 + 16 * i + r;
            if (m < m1) {
                if (wave == 0 && grp == 0) g.mid_scale[(int64_t)(n0 / 128) * g.ld_mid_scale + m] = f.scale;
                // Rows of whole blocks, zero past I.
                *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(g.C) + (int64_t)m * g.sc_m + n0 + wave * 16 + 4 * grp) =
                    cvt4_fp8(f(acc[0][i][0]), f(acc[0][i][1]), f(acc[0][i][2]), f(acc[0][i][3]));
            }
        }
    } else {
        using TC = typename C::TC;
        const int c = n0 + wave * 16 + 4 * grp;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = m0 + 16 * i + r;
            if (m >= m1) continue;
            float f = 1.0f;
            if constexpr (MODE == FP8_DOWN) f = g.row_weight[m];
            TC v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = (TC)(acc[0][i][q] * f);
            TC* out = static_cast<TC*>(g.C) + (int64_t)m * g.sc_m + c;
            if (c + 4 <= g.N) __builtin_memcpy(out, v, sizeof(v));
            else
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (c + q < g.N) out[q] = v[q];
        }
    }
}

template <class C> static int run_wide(const Fp8Gemm& g, hipStream_t stream) {
    const int64_t tiles_n = ((int64_t)g.N + 127) / 128;
    const int64_t tiles_m = C::MODE == FP8_DENSE ? ((int64_t)g.M + C::BM - 1) / C::BM : g.max_tiles;
    int64_t n = tiles_m * tiles_n;
    Fp8Split sp{1, nullptr, nullptr};
    // As many parts as fit the CUs at once, of at least two chunks of k each.
    const int64_t kb = ((int64_t)g.K + 127) / 128;
    int64_t parts = C::WGS * device_cus() / n;
    if (parts > kb / (2 * C::KC)) parts = kb / (2 * C::KC);
    if (parts > 16) parts = 16;
    if (parts > 1) {
        const size_t bytes = (size_t)n * parts * C::THREADS * C::NG * C::MT * 16;
        if (bytes < ((size_t)1 << 30) && gemm_sk_workspace(stream, (size_t)n, bytes, &sp.cnt, &sp.slots) == 0) sp.parts = (int)parts;
    }
    n *= sp.parts;
    if (C::MODE != FP8_DENSE) n = (n + 7) / 8 * 8;
    if (n >= ((int64_t)1 << 32) / C::THREADS) return TV_E_UNSUPPORTED;
    hipLaunchKernelGGL((gemm_fp8_wide_kernel<C>), dim3((unsigned)n), dim3(C::THREADS), 0, stream, g, (int)tiles_n, sp);
    return hipGetLastError();
}

template <int MODE, typename TC, bool EXACT, int ROWS> static int wide_rows(const Fp8Gemm& g, hipStream_t stream) {
    const int rows = MODE == FP8_DENSE ? g.M : g.tile_rows;
    if constexpr (MODE != FP8_DENSE)
        if (rows <= 16) return run_wide<Fp8Wide<MODE, TC, EXACT, 1, ROWS>>(g, stream);
    if (rows <= 32) return run_wide<Fp8Wide<MODE, TC, EXACT, 2, ROWS>>(g, stream);
    return run_wide<Fp8Wide<MODE, TC, EXACT, 4, ROWS>>(g, stream);
}
template <int MODE, typename TC, bool EXACT> static int wide(const Fp8Gemm& g, hipStream_t stream) {
    const bool fast = fast_rows(g.A, MODE == FP8_GATE_UP ? g.tokens : g.M, g.sa_m, g.K) && fast_rows(g.W, g.N, g.sw_n, g.K) &&
                      g.sw_e % 16 == 0 && g.sw_g % 16 == 0;
    return fast ? wide_rows<MODE, TC, EXACT, FP8_ALIGNED>(g, stream) : wide_rows<MODE, TC, EXACT, FP8_ANY>(g, stream);
}

int launch_gemm_fp8_wide(const Fp8Gemm& g, int mode, hipStream_t stream) {
    if (mode == FP8_GATE_UP) return wide<FP8_GATE_UP, uint8_t, true>(g, stream);
    if (mode == FP8_DOWN) return g.dtype_c == TV_FLOAT32 ? wide<FP8_DOWN, float, true>(g, stream) : wide<FP8_DOWN, float, false>(g, stream);
    switch (g.dtype_c) {
        case TV_BFLOAT16: return wide<FP8_DENSE, __bf16, false>(g, stream);
        case TV_FLOAT16: return wide<FP8_DENSE, _Float16, false>(g, stream);
        default: return wide<FP8_DENSE, float, true>(g, stream);
    }
}

} // namespace tvk
