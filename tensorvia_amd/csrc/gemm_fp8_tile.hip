// Products of many rows: BM x BN tiles, operands through LDS with direct loads (gemm_dma_impl.h), the block
// scales as in gemm_fp8.hip.
//
//  * A k-tile is 128 codes, one scale block: 128 bytes of a row, so the LDS rows, the swizzle and the loads are those
//    of the other 8-bit product's K-contiguous operands (DmaOperand's layout: chunk c of row r at c ^ ((r >> 1) & 7)).
//  * A wave's tile is FM x FN blocks of 16 x 16.  Per k-tile each block is one matrix instruction into a fresh
//    result and four multiply-adds that bring it, scaled, into the sum.  The result of a row of blocks is scaled while the
//    next row's instructions run: 4 x 4 cycles of vector ALU per 32 cycles of matrix core.
//  * bf16 [4096,4096]x[11008,4096]: 173 to 180 us, 2.1 PFLOP/s (3 rounds of 688 tiles on 256 CUs; single launches between 167
//    and 201), the matrix cores busy for 52 % of the cycles and LDS for 25 %, at 2.0 GHz under the board's power limit: behind a k-tile's barrier its eight waves read their next
//    fragments all at once.  4096 tokens of 64 experts of 1376, k = 8: gate and up 420-440 us, down 310-320.
//  * Scales of A's rows come through LDS beside the codes (one 4-byte direct load per row and k-tile); W's scale is
//    one value per wave and k-tile, held 64 k-tiles at a time in one register across the lanes.
#include "fp8_common.h"
#include "gemm_dma_impl.h"

#include <type_traits>

namespace tvk {

// Direct loads into LDS at m0 + 16 (4) * lane from base + offset + advance, for the k-loop: the descriptor stays the same
// and the k-tile is the scalar advance.  No memory clobber: the loop's LDS reads may move across (they read the other
// stage; barriers order the stages).  Waited for by explicit vmcnt counts.
__device__ inline void dma16(__amdgpu_buffer_rsrc_t r, unsigned m0v, unsigned off, unsigned advance) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0v), "v"(off), "s"(r), "s"(advance) : "m0");
}
__device__ inline void dma4(__amdgpu_buffer_rsrc_t r, unsigned m0v, unsigned off, unsigned advance) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(m0v), "v"(off), "s"(r), "s"(advance) : "m0");
}

// Buffer descriptor in scalar registers (its values are workgroup-uniform; see DmaOperand::rsrc).
__device__ inline __amdgpu_buffer_rsrc_t uniform_rsrc(const void* p, int64_t bytes) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    const uint64_t v = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)u) |
                       (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32)) << 32;
    const int nr = __builtin_amdgcn_readfirstlane((int)(bytes < 0x7fffffff ? bytes : 0x7fffffff));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(v), (short)0, nr, 0x00020000);
}

template <int MODE_, typename TC_, int BM_, int BN_, int WM_, int WN_, bool EXACT_ = __is_same(TC_, float)> struct Fp8Tile {
    using TC = TC_;
    static constexpr int MODE = MODE_, BM = BM_, BN = BN_, WAVES_M = WM_, WAVES_N = WN_;
    static constexpr bool EXACT = EXACT_; // exact products of a block (mfma_fp8_exact)
    static constexpr int NW = WM_ * WN_, THREADS = NW * 64;
    static constexpr int FM = BM / (16 * WM_), FN = BN / (16 * WN_);
    static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW; // 1 KB loads per wave and k-tile
    static constexpr int ABYTES = BM * 128, BBYTES = BN * 128, SBYTES = NW * 256; // a scale per thread
    static constexpr int STAGES = 2;
    static constexpr bool SPLIT = MODE_ == FP8_DENSE && BM_ == 128; // few tiles: parts of k
    static constexpr int LDS = STAGES * (ABYTES + BBYTES + SBYTES);
    static constexpr int NCOLS = MODE == FP8_GATE_UP ? BN / 2 : BN; // output columns of a tile
    static_assert(PA * 8 * NW == BM && PB * 8 * NW == BN && BM <= THREADS, "loads divide over the waves");
};

// Output columns of the tile, 16 bytes per lane: a wave's rows go through its own part of LDS.
template <class C, typename TS, typename F>
__device__ inline void store_rows(const f32x4 (&acc)[C::FM][C::FN], char* area, char* out, int64_t row_bytes,
                                  int rows, int cols, int lane, const F& value) {
    constexpr int CW = C::FN * 16;                   // columns of the wave
    constexpr int PITCH = CW * (int)sizeof(TS) + 16; // bytes of a staged row
    constexpr int RP = sizeof(TS) == 4 ? 16 : 32;    // rows per pass
    constexpr int CPR = CW * (int)sizeof(TS) / 16;   // chunks of a row
    constexpr int VEC = 16 / (int)sizeof(TS);
    const int r = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int p = 0; p < C::FM * 16 / RP; ++p) {
#pragma unroll
        for (int i = 0; i < RP / 16; ++i)
#pragma unroll
            for (int j = 0; j < C::FN; ++j) {
                TS v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = (TS)value(acc[p * (RP / 16) + i][j][q], p * (RP / 16) + i);
                __builtin_memcpy(area + (16 * i + r) * PITCH + (16 * j + 4 * grp) * (int)sizeof(TS), v, sizeof(v));
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < RP * CPR / 64; ++s) {
            const int id = s * 64 + lane, row = id / CPR, c = (id % CPR) * VEC;
            const u32x4 v = *reinterpret_cast<const u32x4*>(area + row * PITCH + c * (int)sizeof(TS));
            const int m = p * RP + row;
            if (m < rows) {
                char* dst = out + (int64_t)m * row_bytes + c * (int)sizeof(TS);
                if (c + VEC <= cols) {
                    __builtin_memcpy(dst, &v, 16);
                } else {
                    for (int q = 0; q < VEC; ++q)
                        if (c + q < cols) {
                            TS e;
                            __builtin_memcpy(&e, reinterpret_cast<const char*>(&v) + q * sizeof(TS), sizeof(TS));
                            __builtin_memcpy(dst + q * sizeof(TS), &e, sizeof(TS));
                        }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <class C>
__global__ __attribute__((amdgpu_flat_work_group_size(C::THREADS, C::THREADS), amdgpu_waves_per_eu(2, 2)))
void gemm_fp8_tile_kernel(Fp8Gemm g, int tiles_m, int tiles_n, int group_m, Fp8Split sp) {
    __shared__ __attribute__((aligned(1024))) char L[C::LDS];
    constexpr int MODE = C::MODE;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WAVES_N, wn = wave % C::WAVES_N;
    const int r = lane & 15, grp = lane >> 4;

    // Workgroups are dealt round-robin over the 8 XCDs: each takes a contiguous run of the tiles, which share operands in
    // its L2.  (Workgroups that stay for many tiles, the next one's first loads on their way while this one is stored, were
    // slower for the experts, down product 445 us against 354: loads and stores retire in one order, so the next tile's
    // first k-tile waited for the last one's stores.)
    struct Place {
        int m0, m1, n0, expert, id;
    } at;
    int t0 = 0, kt = (g.K + 127) / 128, part = 0; // k-tiles [t0, kt) of this workgroup
    if constexpr (MODE == FP8_DENSE) {
        int bid = blockIdx.x;
        if ((gridDim.x & 7) == 0) bid = (bid & 7) * ((int)gridDim.x >> 3) + (bid >> 3);
        part = bid % sp.parts; // a tile's parts side by side
        bid /= sp.parts;
        int b, tm, tn;
        mfma_tile_of(bid, tiles_m, tiles_n, group_m, b, tm, tn);
        at = Place{tm * C::BM, min(g.M, (tm + 1) * C::BM), tn * C::BN, 0, bid};
        const int all = kt;
        t0 = (int)((int64_t)all * part / sp.parts);
        kt = (int)((int64_t)all * (part + 1) / sp.parts);
    } else {
        const int total = *g.ntiles * tiles_n, per = (total + 7) >> 3; // the grid holds as many as there can be
        const int id = ((int)blockIdx.x >> 3) < per ? ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3) : total;
        if (id >= total) return;
        const int tile = id / tiles_n;
        const int4 e = g.tiles[tile];
        at = Place{e.y, e.z, (id - tile * tiles_n) * C::NCOLS, e.x, id};
    }
    const int k_end = min(g.K, kt * 128);

    // Loads.  Block `blk` of 1 KB is 8 rows; lane l holds chunk l % 8 (swizzled) of row l / 8: its k is kc in blocks of even
    // number and kc ^ 64 in odd ones.
    const unsigned L0 = (unsigned)(uintptr_t)(lds_void*)L;
    const int kc = ((lane & 7) ^ (lane >> 4)) * 16;
    const int wrow = MODE == FP8_GATE_UP ? wn * (C::FN / 2) * 16 : wn * C::FN * 16;
    unsigned aoff[C::PA], boff[C::PB], soff; // soff: the scale of the tile's row threadIdx.x
    __amdgpu_buffer_rsrc_t ra, rb, rs;
    float ws0, ws1; // W's scales: lane l holds k-tile 64 q + l's
    auto load_ws = [&](int t) {
        const int n = at.n0 + (MODE == FP8_GATE_UP ? 0 : wrow);
        const float* row = g.w_scale + (int64_t)at.expert * g.sws_e + (int64_t)(n / 128) * g.sws_n;
        const bool in = n < g.N && t + lane < kt;
        ws0 = in ? row[(int64_t)(t + lane) * g.sws_k] : 0.0f;
        ws1 = MODE == FP8_GATE_UP && in ? row[g.sws_g + (int64_t)(t + lane) * g.sws_k] : 0.0f;
    };
    // Waited for where no other load is on its way: at their uses, behind the next loads, a wait would take those in too.
    auto wait_ws = [&]() { asm volatile("s_waitcnt vmcnt(0)" : "+v"(ws0), "+v"(ws1)); };
    auto setup = [&]() {
#pragma unroll
        for (int j = 0; j < C::PA; ++j) {
            const int blk = wave * C::PA + j, row = blk * 8 + (lane >> 3), k = kc ^ ((blk & 1) * 64);
            const bool in = at.m0 + row < at.m1;
            if constexpr (MODE == FP8_GATE_UP) aoff[j] = in ? (unsigned)(g.row_token[at.m0 + row] * g.sa_m) + k : kOOB;
            else aoff[j] = in ? (unsigned)(row * g.sa_m) + k : kOOB;
        }
#pragma unroll
        for (int j = 0; j < C::PB; ++j) {
            const int blk = wave * C::PB + j, row = blk * 8 + (lane >> 3), k = kc ^ ((blk & 1) * 64);
            if constexpr (MODE == FP8_GATE_UP) {
                const int half = row / C::NCOLS, n = row % C::NCOLS; // gate rows, then up rows
                boff[j] = at.n0 + n < g.N ? (unsigned)(half * g.sw_g + n * g.sw_n) + k : kOOB;
            } else {
                boff[j] = at.n0 + row < g.N ? (unsigned)(row * g.sw_n) + k : kOOB;
            }
        }
        soff = kOOB;
        if (at.m0 + (int)threadIdx.x < at.m1 && (int)threadIdx.x < C::BM) {
            if constexpr (MODE == FP8_GATE_UP) soff = (unsigned)(g.row_token[at.m0 + threadIdx.x] * g.sas_m * 4);
            else soff = (unsigned)((int)threadIdx.x * g.sas_m * 4);
        }
        ra = uniform_rsrc(MODE == FP8_GATE_UP ? g.A : g.A + (int64_t)at.m0 * g.sa_m, 0x7fffffff);
        rb = uniform_rsrc(g.W + (int64_t)at.expert * g.sw_e + (int64_t)at.n0 * g.sw_n, 0x7fffffff);
        rs = uniform_rsrc(MODE == FP8_GATE_UP ? g.a_scale : g.a_scale + (int64_t)at.m0 * g.sas_m, 0x7fffffff);
        load_ws(t0);
        // The descriptors were written by v_readfirstlane: 5 wait states before a load reads them.
        asm volatile("s_nop 4" ::"s"(ra), "s"(rb), "s"(rs));
    };
    constexpr int LD = C::PA + C::PB;
    // Load u of this wave for k-tile t into stage st; chunks past K (in the last k-tile, and all of those behind it) read
    // zeros.
    auto issue_one = [&](int u, int t, int st) {
        const int rem = k_end - t * 128, blk = u < C::PA ? wave * C::PA + u : wave * C::PB + u - C::PA;
        const bool in = (blk & 1 ? kc ^ 64 : kc) < rem;
        if (u < C::PA) dma16(ra, L0 + st * C::ABYTES + blk * 1024, in ? aoff[u] : kOOB, (unsigned)t * 128);
        else dma16(rb, L0 + C::STAGES * C::ABYTES + st * C::BBYTES + blk * 1024, in ? boff[u - C::PA] : kOOB, (unsigned)t * 128);
    };
    auto issue_scales = [&](int t, int st) {
        dma4(rs, L0 + C::STAGES * (C::ABYTES + C::BBYTES) + st * C::SBYTES + wave * 256, t < kt ? soff : kOOB, (unsigned)t * (unsigned)(g.sas_k * 4));
    };

    // Fragment addresses: rows w0 + 16 f + r, chunks grp and grp + 4; rows are instruction offsets.
    const unsigned xa = L0 + kc_off(wm * C::FM * 16 + r, grp);
    const unsigned xb = L0 + C::STAGES * C::ABYTES + kc_off(wrow + r, grp);
    typedef const __attribute__((address_space(3))) char lds_cchar;
    auto frag = [&](unsigned x, int off) {
        const u32x4 lo = *(const __attribute__((address_space(3))) u32x4*)((lds_cchar*)(uintptr_t)x + off);
        const u32x4 hi = *(const __attribute__((address_space(3))) u32x4*)((lds_cchar*)(uintptr_t)(x ^ 64u) + off);
        return join(lo, hi);
    };
    auto bfrag = [&](unsigned x, int j) {
        constexpr int H = C::FN / 2;
        return frag(x, MODE == FP8_GATE_UP ? (j % H) * 2048 + (j / H) * (C::NCOLS * 128) : j * 2048);
    };

    f32x4 acc[C::FM][C::FN];
    // One k-tile, all of whose loads have landed, its first fragments read.  Row i's instructions run while row i - 1's
    // results are scaled into the sums (the last row's in the next k-tile's first).  Before the last row: the next
    // k-tile has landed (it was issued a k-tile ago), every wave has read its last fragment of this one, so behind the
    // barrier the next fragments are read and the loads of the k-tile after it go out, a few beside each row.
    constexpr int SLOT = C::FM >= 8 ? (LD + 3) / 4 : (LD + 2) / 3; // loads per row
    i32x8 fb[C::FN], fa[2];
    f32x4 res[C::FN];
    auto row_scale = [&](int st, int i) {
        return ((const __attribute__((address_space(3))) float*)(uintptr_t)(L0 + C::STAGES * (C::ABYTES + C::BBYTES) + st * C::SBYTES))[wm * C::FM * 16 + 16 * i + r];
    };
    setup();
#pragma unroll
    for (int u = 0; u < LD; ++u) issue_one(u, t0, 0);
    issue_scales(t0, 0);
    float s_gate = 0.0f, s_up = 0.0f; // scales of the row in res
#pragma unroll
    for (int j = 0; j < C::FN; ++j) res[j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
        for (int j = 0; j < C::FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    wait_ws();
    wait_vmcnt<0>();
    dma_barrier();
#pragma unroll
    for (int u = 0; u < SLOT; ++u) issue_one(u, t0 + 1, 1);
    issue_scales(t0 + 1, 1);
    // A wave none of whose rows are in the tile only loads and keeps step.
    const bool idle = MODE != FP8_DENSE && at.m0 + wm * C::FM * 16 >= at.m1;
    if (idle) {
        for (int t = t0; t < kt; ++t) {
            const int st = (t - t0) & 1;
#pragma unroll
            for (int u = SLOT; u < LD; ++u) issue_one(u, t + 1, st ^ 1);
            wait_vmcnt<0>();
            dma_barrier();
#pragma unroll
            for (int u = 0; u < SLOT; ++u) issue_one(u, t + 2, st);
            issue_scales(t + 2, st);
        }
    } else {
#pragma unroll
        for (int j = 0; j < C::FN; ++j) fb[j] = bfrag(xb, j);
        fa[0] = frag(xa, 0);
        float s_row = row_scale(0, 0); // of the row in fa
        for (int t = t0; t < kt; ++t) {
            const int turn = t - t0;
            if ((turn & 63) == 0 && turn > 0) {
                load_ws(t);
                wait_ws();
            }
            const int st = turn & 1;
            const unsigned xa_t = xa + st * C::ABYTES, xa_n = xa + (st ^ 1) * C::ABYTES, xb_n = xb + (st ^ 1) * C::BBYTES;
            const float w0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ws0), turn & 63));
            const float w1 = MODE == FP8_GATE_UP ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ws1), turn & 63)) : w0;
#pragma unroll
            for (int i = 0; i < C::FM; ++i) {
                const bool last = i == C::FM - 1;
                if (last) {
                    wait_vmcnt<0>();
                    dma_barrier();
                }
                // Loads: slot 0 beside the last row (k-tile t + 2 into this stage), then beside rows 0, 1, ... (t + 1).
                const int slot = last ? 0 : i + 1;
#pragma unroll
                for (int u = slot * SLOT; u < (slot + 1) * SLOT && u < LD; ++u) issue_one(u, last ? t + 2 : t + 1, last ? st : st ^ 1);
                if (last) issue_scales(t + 2, st);
                float s_next = 0.0f;
                if (!last) {
                    s_next = row_scale(st, i + 1);
                    fa[(i + 1) & 1] = frag(xa_t, (i + 1) * 2048);
                }
                const int p = i == 0 ? C::FM - 1 : i - 1; // the row in res
#pragma unroll
                for (int j = 0; j < C::FN; ++j) {
                    const float s = MODE == FP8_GATE_UP && j >= C::FN / 2 ? s_up : s_gate;
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[p][j][q] = __builtin_fmaf(s, res[j][q], acc[p][j][q]);
                    if constexpr (C::EXACT) res[j] = mfma_fp8_exact(fb[j], fa[i & 1]);
                    else res[j] = mfma_fp8(fb[j], fa[i & 1]);
                    if (last) fb[j] = bfrag(xb_n, j);
                }
                if (last) {
                    s_next = row_scale(st ^ 1, 0);
                    fa[0] = frag(xa_n, 0);
                }
                s_gate = s_row * w0;
                s_up = s_row * w1;
                s_row = s_next;
                // The order above, row by row: left to itself the scheduler brings the reads of several rows forward and runs out
                // of registers.
                if constexpr (!C::EXACT) {
                    if (!last) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 3, 0);
#pragma unroll
                    for (int j = 0; j < C::FN; ++j) {
                        __builtin_amdgcn_sched_group_barrier(SG_VALU, 4, 0);
                        __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
                        if (last) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 2, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int j = 0; j < C::FN; ++j) {
            const float s = MODE == FP8_GATE_UP && j >= C::FN / 2 ? s_up : s_gate;
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[C::FM - 1][j][q] = __builtin_fmaf(s, res[j][q], acc[C::FM - 1][j][q]);
        }
    }
    wait_vmcnt<0>(); // the loads past the end have landed
    dma_barrier();   // every wave is done with the k-tiles: LDS is free

    const int m0 = at.m0, m1 = at.m1, n0 = at.n0, bid = at.id;
    char* const a1 = L;                           // A's stages
    char* const b1 = L + C::STAGES * C::ABYTES;   // W's
    const int mw = m0 + wm * C::FM * 16; // first row of the wave
    if constexpr (MODE == FP8_DENSE) {
        if (C::SPLIT && sp.parts > 1) {
            // Partial sums in register order, a slot per part; the last part to arrive sums them in part order.
            constexpr int BYTES = C::THREADS * C::FM * C::FN * 16;
            const __amdgpu_buffer_rsrc_t slots = make_rsrc(sp.slots + (int64_t)bid * sp.parts * BYTES, (int64_t)sp.parts * BYTES);
            int* last = reinterpret_cast<int*>(L);
            const int lane16 = (int)threadIdx.x * 16;
#pragma unroll
            for (int i = 0; i < C::FM; ++i)
#pragma unroll
                for (int j = 0; j < C::FN; ++j) slot_store16(slots, part * BYTES + (i * C::FN + j) * C::THREADS * 16 + lane16, acc[i][j]);
            publish_and_count(sp.cnt + bid, sp.parts, last);
            const bool mine = *last;
            __syncthreads(); // the flag is read: LDS is free again
            if (!mine) return;
#pragma unroll
            for (int i = 0; i < C::FM; ++i)
#pragma unroll
                for (int j = 0; j < C::FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
            for (int q = 0; q < sp.parts; ++q)
#pragma unroll
                for (int i = 0; i < C::FM; ++i)
#pragma unroll
                    for (int j = 0; j < C::FN; ++j) acc[i][j] += slot_load16<f32x4>(slots, q * BYTES + (i * C::FN + j) * C::THREADS * 16 + lane16);
            slot_count_reset(sp.cnt + bid);
        }
        using TC = typename C::TC;
        char* area = L + wave * (C::LDS / C::NW / 1024 * 1024);
        const int nw = n0 + wrow;
        char* out = static_cast<char*>(g.C) + ((int64_t)mw * g.sc_m + nw) * (int64_t)sizeof(TC);
        store_rows<C, TC>(acc, area, out, g.sc_m * (int64_t)sizeof(TC), m1 - mw, g.N - nw, lane, [](float v, int) { return v; });
    } else if constexpr (MODE == FP8_DOWN) {
        // Rows of y as f16 beside a power of two per row and 64 columns (experts_sum_kernel multiplies them back).
        constexpr int CW = C::FN * 16;
        static_assert(CW == 64, "a scale per 64 columns");
        const int nw = n0 + wrow;
        float inv[C::FM], wt[C::FM];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) wt[i] = mw + 16 * i + r < m1 ? g.row_weight[mw + 16 * i + r] : 0.0f;
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const int m = mw + 16 * i + r;
            const float w = wt[i];
            unsigned mx = 0;
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[i][j][q] *= w;
                    const unsigned b = abs_bits(acc[i][j][q]);
                    mx = umax(mx, b < 0x7f800000u ? b : 0u);
                }
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 16));
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 32));
            // 2^e, the largest value's exponent held to [-126, 126] so that the inverse is a normal number too.
            int e = (int)(mx >> 23) - 127;
            e = e < -126 ? -126 : e > 126 ? 126 : e;
            inv[i] = __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
            if (grp == 0 && m < m1 && nw < g.N) g.row_scale[(int64_t)m * g.ld_row_scale + nw / 64] = __builtin_bit_cast(float, (unsigned)(127 + e) << 23);
        }
        char* area = L + wave * (C::LDS / C::NW / 1024 * 1024);
        char* out = static_cast<char*>(g.C) + ((int64_t)mw * g.sc_m + nw) * 2;
        store_rows<C, _Float16>(acc, area, out, g.sc_m * 2, m1 - mw, (int)g.sc_m - nw, lane, [&](float v, int i) { return v * inv[i]; });
    } else {
        // silu(gate) * up, and its codes: the tile's 128 columns are one block of each row.
        constexpr int H = C::FN / 2;
        static_assert(C::NCOLS == 128, "a tile is one block of its rows");
        unsigned* most = reinterpret_cast<unsigned*>(b1); // [BM][WAVES_N]
        // [BM] rows of 128 bytes, 16-byte chunk c of row m at c ^ (m & 7): a wave writes one column of words of 16 rows.
        char* codes = a1;
        static_assert(C::BM * C::WAVES_N * 4 <= C::BBYTES, "LDS");
        const ActCoef silu = act_coef(TV_ACT_SILU);
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            unsigned mx = 0;
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[i][j][q] = act_logistic(acc[i][j][q], silu) * acc[i][j + H][q];
                    mx = umax(mx, abs_bits(acc[i][j][q]));
                }
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 16));
            mx = umax(mx, (unsigned)__shfl_xor((int)mx, 32));
            if (grp == 0) most[(wm * C::FM * 16 + 16 * i + r) * C::WAVES_N + wn] = mx;
        }
        dma_barrier();
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const int row = wm * C::FM * 16 + 16 * i + r;
            unsigned mx = 0;
#pragma unroll
            for (int w = 0; w < C::WAVES_N; ++w) mx = umax(mx, most[row * C::WAVES_N + w]);
            const Fp8Block f = fp8_block(mx);
            if (wn == 0 && grp == 0 && m0 + row < m1) g.mid_scale[(int64_t)(n0 / 128) * g.ld_mid_scale + m0 + row] = f.scale;
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const f32x4 v = acc[i][j];
                *reinterpret_cast<unsigned*>(codes + row * 128 + (((wrow / 16 + j) ^ (row & 7)) << 4) + 4 * grp) =
                    cvt4_fp8(f(v[0]), f(v[1]), f(v[2]), f(v[3]));
            }
        }
        dma_barrier();
        uint8_t* out = static_cast<uint8_t*>(g.C) + (int64_t)m0 * g.sc_m + n0;
        for (int id = threadIdx.x; id < C::BM * 8; id += C::THREADS) {
            const int row = id >> 3, c = (id & 7) * 16;
            if (m0 + row < m1) *reinterpret_cast<u32x4*>(out + (int64_t)row * g.sc_m + c) = *reinterpret_cast<const u32x4*>(codes + row * 128 + (((id & 7) ^ (row & 7)) << 4));
        }
    }
}

// The loaders add 32-bit offsets to a tile's base (for gathered rows the operand's), which stay below 2^31 - 2^20.  Among them are those
// of the two k-tiles that the loop asks for past the end: their lanes are out of range, but the range check subtracts the
// k-tile's scalar advance from the descriptor's size, so an advance beyond the size would let them through.
bool fp8_tile_ok(const Fp8Gemm& g, int mode) {
    const int64_t lim = ((int64_t)1 << 31) - ((int64_t)1 << 20);
    const int64_t a_rows = mode == FP8_GATE_UP ? g.tokens : 256;
    const int64_t w_off = (mode == FP8_GATE_UP ? g.sw_g : 0) + 256 * g.sw_n + g.K;
    return fast_rows(g.A, g.M, g.sa_m, g.K) && fast_rows(g.W, g.N, g.sw_n, g.K) && g.sw_e % 16 == 0 && g.sw_g % 16 == 0 &&
           a_rows * g.sa_m + g.K < lim && a_rows * g.sas_m * 4 + (g.K / 128 + 2) * g.sas_k * 4 < lim && w_off < lim && g.K > 0;
}

// The operands as pad_fp8_operands leaves them, but for their addresses.
static Fp8Gemm padded_fp8(const Fp8Gemm& g, int mode, bool* pad_a, bool* pad_w) {
    const int64_t P = (g.K + 15) / 16 * 16;
    // The down product's rows are this library's own and already padded.
    *pad_a = mode != FP8_DOWN && !fast_rows(g.A, mode == FP8_GATE_UP ? g.tokens : g.M, g.sa_m, g.K);
    *pad_w = !fast_rows(g.W, g.N, g.sw_n, g.K) || g.sw_e % 16 != 0 || g.sw_g % 16 != 0;
    Fp8Gemm p = g;
    if (*pad_a) {
        p.A = nullptr;
        p.sa_m = P;
    }
    if (*pad_w) {
        p.W = nullptr;
        p.sw_n = P;
        p.sw_g = mode == FP8_GATE_UP ? g.N * P : 0;
        p.sw_e = mode == FP8_GATE_UP ? 2 * g.N * P : mode == FP8_DOWN ? g.N * P : 0;
    }
    p.K = (int32_t)P;
    return p;
}

bool fp8_pad_ok(const Fp8Gemm& g, int mode) {
    bool pad_a, pad_w;
    const Fp8Gemm p = padded_fp8(g, mode, &pad_a, &pad_w);
    return fp8_tile_ok(p, mode) && !(pad_w && mode == FP8_GATE_UP && g.experts > 1 && g.sw_e != 2 * g.sw_g);
}

static int64_t pad_a_rows(const Fp8Gemm& g, int mode) { return mode == FP8_GATE_UP ? g.tokens : g.M; }
static int64_t pad_w_rows(const Fp8Gemm& g, int mode) {
    return (mode == FP8_DENSE ? 1 : mode == FP8_GATE_UP ? 2 * (int64_t)g.experts : g.experts) * g.N;
}

Fp8PadBytes fp8_pad_bytes(const Fp8Gemm& g, int mode) {
    bool pad_a, pad_w;
    const Fp8Gemm p = padded_fp8(g, mode, &pad_a, &pad_w);
    return {pad_a ? (size_t)(pad_a_rows(g, mode) * p.K) : 0, pad_w ? (size_t)(pad_w_rows(g, mode) * p.K) : 0};
}

int fp8_pad_buffers(const Fp8PadBytes& bytes, hipStream_t stream, Fp8Pads* pads) {
    *pads = Fp8Pads{};
    if (bytes.w && gemm_pad_workspace(stream, bytes.w, 1, &pads->w) != 0) return TV_E_UNSUPPORTED;
    if (bytes.a && gemm_pad_workspace(stream, bytes.a, 0, &pads->a) != 0) return TV_E_UNSUPPORTED;
    return 0;
}

int pad_fp8_operands(Fp8Gemm& g, int mode, const Fp8Pads& pads, hipStream_t stream) {
    bool pad_a, pad_w;
    Fp8Gemm p = padded_fp8(g, mode, &pad_a, &pad_w);
    const int64_t P = p.K, a_rows = pad_a_rows(g, mode);
    PadJob jobs[2];
    int n = 0;
    if (pad_a) {
        jobs[n++] = PadJob{g.A, pads.a, a_rows, a_rows, g.sa_m, 0, g.K, P};
        p.A = static_cast<const uint8_t*>(pads.a);
    }
    if (pad_w) {
        jobs[n++] = PadJob{g.W, pads.w, g.N, pad_w_rows(g, mode), g.sw_n, mode == FP8_GATE_UP ? g.sw_g : g.sw_e, g.K, P};
        p.W = static_cast<const uint8_t*>(pads.w);
    }
    g = p;
    return n ? launch_pad_rows(jobs, n, 1, stream) : 0;
}

template <class C> static int run_tile(const Fp8Gemm& g, hipStream_t stream) {
    const int64_t tiles_n = (g.N + C::NCOLS - 1) / C::NCOLS;
    const int64_t tiles_m = C::MODE == FP8_DENSE ? (g.M + C::BM - 1) / C::BM : g.max_tiles;
    int64_t n = tiles_m * tiles_n;
    Fp8Split sp{1, nullptr, nullptr};
    if (C::MODE != FP8_DENSE) {
        n = (n + 7) / 8 * 8;
    } else if (C::SPLIT) {
        // Few tiles: as many parts of k as fit the CUs at once, of at least four k-tiles each.
        const int64_t kt = ((int64_t)g.K + 127) / 128;
        int64_t parts = 2 * device_cus() / n;
        if (parts > kt / 4) parts = kt / 4;
        if (parts > 8) parts = 8;
        if (parts > 1) {
            const size_t bytes = (size_t)n * parts * C::BM * C::BN * 4;
            if (gemm_sk_workspace(stream, (size_t)n, bytes, &sp.cnt, &sp.slots) == 0) sp.parts = (int)parts;
        }
        n *= sp.parts;
    }
    if (n >= ((int64_t)1 << 31) / C::THREADS) return TV_E_UNSUPPORTED; // 2^31 threads
    hipLaunchKernelGGL((gemm_fp8_tile_kernel<C>), dim3((unsigned)n), dim3(C::THREADS), 0, stream, g, (int)tiles_m, (int)tiles_n, 4, sp);
    return hipGetLastError();
}

int launch_gemm_fp8_tile(const Fp8Gemm& g, int mode, hipStream_t stream) {
    if (mode == FP8_GATE_UP && g.exact) return run_tile<Fp8Tile<FP8_GATE_UP, uint8_t, 128, 256, 2, 4, true>>(g, stream);
    if (mode == FP8_GATE_UP) return g.tile_rows == 256 ? run_tile<Fp8Tile<FP8_GATE_UP, uint8_t, 256, 256, 2, 4>>(g, stream)
                                                       : run_tile<Fp8Tile<FP8_GATE_UP, uint8_t, 128, 256, 2, 4>>(g, stream);
    if (mode == FP8_DOWN) return g.tile_rows == 256 ? run_tile<Fp8Tile<FP8_DOWN, _Float16, 256, 256, 2, 4>>(g, stream)
                                                    : run_tile<Fp8Tile<FP8_DOWN, _Float16, 128, 256, 2, 4>>(g, stream);
    const bool big = g.tile_rows == 256;
    switch (g.dtype_c) {
        case TV_BFLOAT16: return big ? run_tile<Fp8Tile<FP8_DENSE, __bf16, 256, 256, 2, 4>>(g, stream) : run_tile<Fp8Tile<FP8_DENSE, __bf16, 128, 128, 2, 2>>(g, stream);
        case TV_FLOAT16: return big ? run_tile<Fp8Tile<FP8_DENSE, _Float16, 256, 256, 2, 4>>(g, stream) : run_tile<Fp8Tile<FP8_DENSE, _Float16, 128, 128, 2, 2>>(g, stream);
        default: return run_tile<Fp8Tile<FP8_DENSE, float, 128, 128, 2, 2>>(g, stream);
    }
}

} // namespace tvk
