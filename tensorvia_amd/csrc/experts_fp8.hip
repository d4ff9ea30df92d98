// A layer of experts on quantised rows: plan, gate-and-up product, quantisation, down product, sum over slots.
#include "fp8_common.h"

#include <type_traits>

namespace tvk {

// The plan orders the slots (t, j) by expert, in rising slot order within one, and cuts each expert's rows into
// tiles of `bm`.  Its integers, in the workspace:
//   ntiles  [1], tiles [max_tiles][4]   expert, first row and last row + 1 of each tile
//   row_token [TK], row_weight [TK]     token of a row, and its routing weight
//   slot_row [TK]                       row of a slot, -1 for a slot without expert
// Every workgroup reads all ids (they come from L2) and counts, per expert, the slots before its own run and those
// from there on (LDS atomics on counts, whose order does not matter); the sums over experts give every expert's first
// row, so no workgroup waits for another.  Each wave of it then places its part of the run 64 slots at a time: lanes
// with the same expert find each other by one ballot per bit of the id, so their order is the slots'.
// 512 slots take 4.1 us, 32768 8.7.  (One workgroup for all slots took 59 us for 32768: 32 dependent rounds a wave.)
constexpr int kPlanWaves = 16, kPlanThreads = 64 * kPlanWaves;
constexpr int kPlanRounds = 2;                                // rounds of 64 slots a wave places
constexpr int kPlanSlots = kPlanThreads * kPlanRounds;        // slots of a workgroup
static_assert(kPlanThreads >= TV_ROUTE_MAX_EXPERTS, "a thread per expert");

__global__ __launch_bounds__(kPlanThreads) void expert_plan_kernel(const int* ids, const float* weights, int tk, int E, int k, int bm,
                                                                   int* ntiles, int4* tiles, float* row_weight,
                                                                   int* row_token, int* slot_row) {
    __shared__ int before[TV_ROUTE_MAX_EXPERTS], behind[TV_ROUTE_MAX_EXPERTS];
    __shared__ int cnt[kPlanWaves][TV_ROUTE_MAX_EXPERTS];
    __shared__ int wave_rows[kPlanWaves], wave_tiles[kPlanWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int start = (int)blockIdx.x * kPlanSlots;
    // The wave's own slots, loaded first.
    int own[kPlanRounds];
    float weight[kPlanRounds];
#pragma unroll
    for (int q = 0; q < kPlanRounds; ++q) {
        const int slot = start + (wave * kPlanRounds + q) * 64 + lane;
        own[q] = slot < tk ? ids[slot] : -1;
        weight[q] = slot < tk ? weights[slot] : 0.0f;
    }
    if (tid < E) {
        before[tid] = behind[tid] = 0;
        for (int w = 0; w < kPlanWaves; ++w) cnt[w][tid] = 0;
    }
    __syncthreads();
    for (int i0 = 0; i0 < tk; i0 += 8 * kPlanThreads) { // eight loads in flight
        int e[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * kPlanThreads + tid;
            e[u] = i < tk ? ids[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if ((unsigned)e[u] < (unsigned)E) atomicAdd(i0 + u * kPlanThreads + tid < start ? &before[e[u]] : &behind[e[u]], 1);
    }
#pragma unroll
    for (int q = 0; q < kPlanRounds; ++q)
        if ((unsigned)own[q] < (unsigned)E) atomicAdd(&cnt[wave][own[q]], 1);
    __syncthreads();
    // Thread e: expert e's rows, the sums over the experts before it, and the first row of each wave's slots.
    const int rows = tid < E ? before[tid] + behind[tid] : 0, nt = (rows + bm - 1) / bm;
    int r_incl = rows, t_incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int a = __shfl_up(r_incl, d), b = __shfl_up(t_incl, d);
        if (lane >= d) {
            r_incl += a;
            t_incl += b;
        }
    }
    if (lane == 63) {
        wave_rows[wave] = r_incl;
        wave_tiles[wave] = t_incl;
    }
    __syncthreads();
    if (tid < E) {
        int r0 = r_incl - rows, t0 = t_incl - nt;
        for (int w = 0; w < wave; ++w) {
            r0 += wave_rows[w];
            t0 += wave_tiles[w];
        }
        if (blockIdx.x == 0) {
            for (int i = 0; i < nt; ++i) tiles[t0 + i] = int4{tid, r0 + i * bm, r0 + min(rows, (i + 1) * bm), 0};
            if (tid == E - 1) *ntiles = t0 + nt;
        }
        int row = r0 + before[tid];
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = cnt[w][tid];
            cnt[w][tid] = row;
            row += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPlanRounds; ++q) {
        const int slot = start + (wave * kPlanRounds + q) * 64 + lane, e = own[q];
        const bool has = (unsigned)e < (unsigned)E;
        uint64_t same = __ballot(has);
#pragma unroll
        for (int b = 0; b < 10; ++b) { // TV_ROUTE_MAX_EXPERTS = 2^10
            const bool bit = e >> b & 1;
            const uint64_t set = __ballot(bit);
            same &= bit ? set : ~set;
        }
        if (has) {
            const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
            // Read by every lane of the group before its first lane moves it on (one wave, in order).
            const int row = __hip_atomic_load(&cnt[wave][e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT) + rank;
            row_weight[row] = weight[q];
            row_token[row] = slot / k;
            slot_row[slot] = row;
            if (rank == 0)
                (void)__hip_atomic_fetch_add(&cnt[wave][e], __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        } else if (slot < tk) {
            slot_row[slot] = -1;
        }
    }
}

// C[t] = sum over the token's slots of their rows of y (already times their weights), in slot order.  y is fp32, or f16 beside
// a power of two per row and 64 columns (row_scale).  32768 slots of 4096 columns in f16 (300 MB with the result): 58 us, 5.1 TB/s.
template <typename T, typename Y>
__global__ __launch_bounds__(256) void experts_sum_kernel(const Y* y, int64_t sy, const float* row_scale, int64_t ld, const int* slot_row,
                                                          int64_t tokens, int64_t H, int k, T* C, int64_t sc) {
    const int64_t per = ((H + 7) / 8 + blockDim.x - 1) / blockDim.x;
    for (int64_t i = blockIdx.x; i < tokens * per; i += gridDim.x) {
        const int64_t t = i / per, h = ((i - t * per) * blockDim.x + threadIdx.x) * 8, left = H - h;
        if (left <= 0) continue;
        float sum[8] = {};
        // Eight slots' rows are on their way at once; slots without expert read row 0 and are not used.
        for (int j0 = 0; j0 < k; j0 += 8) {
            int row[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = j0 + j < k ? slot_row[t * k + j0 + j] : -1;
            Eight<Y> v[8];
            float s[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = row[j] < 0 ? 0 : row[j];
                v[j].load(y + r * sy, h, sy); // y's rows are padded to whole chunks
                s[j] = sizeof(Y) == 2 ? row_scale[r * ld + h / 64] : 1.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int q = 0; q < 8; ++q) sum[q] = row[j] < 0 ? sum[q] : sum[q] + (sizeof(Y) == 2 ? (float)v[j].e[q] * s[j] : (float)v[j].e[q]);
        }
        store8(C + t * sc + h, left, sum);
    }
}

// The scratch of one call, carved from the workspace.
struct ExpertScratch {
    int *ntiles, *row_token, *slot_row;
    int4* tiles;
    float* row_weight;
    float* mid;       // inner rows in fp32 (few rows), [rows][ipad]
    uint8_t* codes;   // inner rows quantised, [rows][ipad]
    float* mid_scale; // [I / 128][rows]
    void* y;          // slots' products, [rows][hpad]: fp32 (few rows) or f16 with
    float* row_scale; // [rows][ld]
};

// Rows per expert (on average) from which the products take tiles through LDS, and tiles of 256 rows instead of 128.  us on
// tiles / without, 64 experts of 1376, k = 8, tiles without exact sums: 20 rows 272 / 257, 25 rows 277 / 297; with exact sums: 24 rows 298 /
// 262, 28 rows 286 / 304.  Where tiles need the weights in padded rows, copied on every call, from more: [T,4095], 64 experts of 1377, 64
// rows 735 / 583, 96 rows 734 / 700, 128 rows 744 / 872; W2 alone, [T,2048], 16 experts of 1001, 75 rows 64 / 66.  64 rows: 333 in
// tiles of 256, 338 of 128.
constexpr int kTileRows = 22, kExactTileRows = 28, kPadTileRows = 100, kPadDownTileRows = 72, kBigTileRows = 64;
// Slots from which tiles with a bf16 result go without exact sums.  A moved code of a row's largest value changes its result by a
// fourteenth, and with few rows a few of them decide the error: relative to the plain form's, over 40 calls each of 8 experts, median and
// largest, I 128 / H 512 and I 512 / H 1536: 240 slots 1.12, 4.3 and 1.24, 2.9; 1000 slots 1.18, 2.3 and 1.21, 1.8; 5600
// slots 1.22, 1.5 and 1.24, 1.32; 11200 slots 1.25, 1.42 and 1.24, 1.34.  Exact sums below that: us, exact / not, [T,4096], 64 experts
// of 1376, k = 8: 256 tokens 290 / 274, 512 367 / 324, 1000 444 / 388; [T,1024], 8 of 512, k = 2: 110 tokens 25 / 29, 1500 42 / 47;
// [4000,4096], 8 of 1376, k = 2: 303 / 226.
constexpr int kExactSlots = 8192;
// Below those, workgroups of 128 columns read an expert's weights once for up to 64 rows, workgroups of 16 columns and 16
// rows read them for every 16 rows but are eight times as many.  The first run where at most one workgroup per expert
// and 128 of I makes at least kWideGroups, or with more than kWideRows rows an expert more than kSomeGroups.  us, wide /
// direct, [tokens, H, I, E, k]: [20,4096,640,60,4] (300 workgroups) 93 / 100; [30,4096,200,64,4] (128, 1.9 rows) 54 / 64;
// [30,2048,1024,16,4] (128, 7.5 rows) 34 / 36, 100 tokens (25 rows) 41 / 56; [32,4096,1376,8,2] (88, 8 rows) 48 / 45, 64 tokens (16
// rows) 50 / 55; [100,1003,503,16,4] (64, 25 rows) 37 / 35; [110,1024,512,8,2] (32, 27 rows) 27 / 23.
constexpr int kWideGroups = 128, kSomeGroups = 64, kWideRows = 13;

// Workgroups of the tiles' and the wide kernels' grids, 512 threads each.
constexpr int64_t kTileGrid = (int64_t)1 << 22, kWideGrid = (int64_t)1 << 23;

// Tokens up to which their slots may go without a plan.
constexpr int kFewTokens = 4;

static int run_experts(const tv_experts_fp8_args& a, hipStream_t stream) {
    const int tk = (int)(a.T * a.k);
    const int64_t hb = (a.H + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK, ib = (a.I + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK;
    const int64_t ipad = ib * TV_FP8_BLOCK, hpad = (a.H + 7) / 8 * 8, ld = (a.H + 63) / 64;

    Fp8Gemm up{};
    up.M = (int)a.T;
    up.tokens = (int)a.T;
    up.experts = a.E;
    up.A = static_cast<const uint8_t*>(a.A);
    up.sa_m = a.sa_m;
    up.a_scale = a.a_scale; up.sas_m = a.sas_m; up.sas_k = a.sas_k;
    up.W = static_cast<const uint8_t*>(a.W1);
    up.sw_e = a.sw1_e; up.sw_g = a.sw1_g; up.sw_n = a.sw1_n;
    up.w_scale = a.w1_scale;
    up.sws_e = 2 * ib * hb; up.sws_g = ib * hb; up.sws_n = hb; up.sws_k = 1;
    up.N = (int)a.I; up.K = (int)a.H;
    Fp8Gemm down = up;
    down.M = tk;
    down.sa_m = ipad;
    down.A = nullptr;
    down.sas_m = 1; down.sas_k = tk;
    down.W = static_cast<const uint8_t*>(a.W2);
    down.sw_e = a.sw2_e; down.sw_g = 0; down.sw_n = a.sw2_n;
    down.w_scale = a.w2_scale;
    down.sws_e = hb * ib; down.sws_g = 0; down.sws_n = ib; down.sws_k = 1;
    down.N = (int)a.H; down.K = (int)a.I;

    // A few tokens, whose slots rarely share an expert: no plan, a slot a row, two launches (4 tokens, 64 experts of 1376, k = 8:
    // 99 us, 108 with plan, quantisation and sum as launches of their own; 8 tokens of 64 experts of 256, k = 4: 49, 37).
    down.slots = up.slots = a.k;
    down.ids = up.ids = a.ids;
    down.route_w = a.weights;
    down.dtype_c = a.dtype_c;
    if ((a.T == 1 || (a.T <= kFewTokens && 2 * tk <= a.E)) && a.I > 0 && fp8_token_ok(down, (int)a.T)) {
        void* mid = nullptr;
        const int rc = experts_workspace(stream, (size_t)tk * ipad * 4, &mid);
        if (rc) return rc;
        Fp8Gemm g = up;
        g.M = tk;
        g.dtype_c = TV_FLOAT32;
        g.C = mid; g.sc_m = ipad;
        const int rc2 = launch_gemm_fp8(g, FP8_SLOT_UP, stream);
        if (rc2) return rc2;
        down.C = a.C; down.sc_m = a.sc_m;
        return launch_gemm_fp8_token(down, static_cast<const float*>(mid), ipad, (int)a.T, stream);
    }

    const bool pad_up = !fp8_tile_ok(up, FP8_GATE_UP), pad_down = !fp8_tile_ok(down, FP8_DOWN);
    // The inner rows are rounded to e4m3: the 8-bit instructions' error of 1.5e-5 moves one value in two thousand to the other code
    // beside it, together 1.2e-3 of the result.  Exact sums cost little where W's bytes bound the call (100 tokens of 8 experts of 1376
    // 56 us, 50 without; 16 of 64 228, 223), but tiles half as much again (4096 tokens 1240 us, 820 without): there bf16 results,
    // whose own rounding is 1.7e-3, go without (2.0e-3 together), and fp16 ones (3.3e-4) do not.
    up.exact = a.dtype_c != TV_BFLOAT16 || tk < kExactSlots;
    bool tiled = tk >= (int64_t)(pad_up ? kPadTileRows : pad_down ? kPadDownTileRows : up.exact ? kExactTileRows : kTileRows) * a.E && a.dtype_c != TV_FLOAT32 && a.I > 0;
    tiled = tiled && (!pad_up || fp8_pad_ok(up, FP8_GATE_UP)) && (!pad_down || fp8_pad_ok(down, FP8_DOWN));
    // Rows of up to `bm` make at most this many tiles.  A grid's threads are limited: calls beyond take the next kernel, the direct one
    // runs in several launches.
    const auto tiles_of = [&](int64_t bm) { return (tk < a.E ? tk : a.E) + tk / bm; };
    const auto grid_ok = [&](int64_t bm, int64_t most) { return tiles_of(bm) * (hb > ib ? hb : ib) <= most - 8; };
    const int tile_rows = tk >= (int64_t)kBigTileRows * a.E && !up.exact ? 256 : 128;
    tiled = tiled && grid_ok(tile_rows, kTileGrid);
    // One buffer holds W1's copy, then W2's.  Without room for it the other kernels run.
    Fp8Pads pads{};
    if (tiled && (pad_up || pad_down)) {
        Fp8PadBytes bytes = pad_up ? fp8_pad_bytes(up, FP8_GATE_UP) : Fp8PadBytes{};
        const size_t w2 = pad_down ? fp8_pad_bytes(down, FP8_DOWN).w : 0;
        bytes.w = bytes.w > w2 ? bytes.w : w2;
        tiled = fp8_pad_buffers(bytes, stream, &pads) == 0;
    }
    const int64_t groups = (int64_t)(tk < a.E ? tk : a.E) * ib;
    const int wide_rows = tk <= 8 * a.E ? 16 : tk <= 24 * a.E ? 32 : 64;
    const bool wide = !tiled && a.I > 0 && (groups >= kWideGroups || (groups > kSomeGroups && tk > kWideRows * a.E)) && grid_ok(wide_rows, kWideGrid);
    const int bm = tiled ? tile_rows : wide ? wide_rows : 16;
    const int max_tiles = (int)tiles_of(bm);

    ExpertScratch s{};
    size_t need = 0;
    char* base = nullptr;
    auto carve = [&]() {
        need = 0;
        auto take = [&](auto*& p, size_t bytes) {
            p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + need);
            need += (bytes + 255) / 256 * 256;
        };
        take(s.ntiles, 4);
        take(s.tiles, (size_t)max_tiles * 16);
        take(s.row_weight, (size_t)tk * 4);
        take(s.row_token, (size_t)tk * 4);
        take(s.slot_row, (size_t)tk * 4);
        if (!tiled && !wide) take(s.mid, (size_t)tk * ipad * 4);
        take(s.codes, (size_t)tk * ipad);
        take(s.mid_scale, (size_t)tk * ib * 4);
        char* y = nullptr;
        take(y, (size_t)tk * hpad * (tiled ? 2 : 4));
        s.y = y;
        if (tiled) take(s.row_scale, (size_t)tk * ld * 4);
    };
    carve();
    void* ws = nullptr;
    int rc = experts_workspace(stream, need, &ws);
    if (rc) return rc;
    base = static_cast<char*>(ws);
    carve();

    hipLaunchKernelGGL(expert_plan_kernel, dim3((tk + kPlanSlots - 1) / kPlanSlots), dim3(kPlanThreads), 0, stream, a.ids, a.weights, tk, a.E, a.k, bm, s.ntiles,
                       s.tiles, s.row_weight, s.row_token, s.slot_row);
    rc = hipGetLastError();
    if (rc) return rc;
    for (Fp8Gemm* g : {&up, &down}) {
        g->row_token = s.row_token;
        g->row_weight = s.row_weight;
        g->tiles = s.tiles;
        g->ntiles = s.ntiles;
        g->max_tiles = max_tiles;
        g->tile_rows = bm;
        g->mid_scale = s.mid_scale; g->ld_mid_scale = tk;
        g->row_scale = s.row_scale; g->ld_row_scale = ld;
    }
    if (tiled) {
        if (pad_up) {
            rc = pad_fp8_operands(up, FP8_GATE_UP, pads, stream);
            if (rc) return rc;
        }
        up.C = s.codes; up.sc_m = ipad;
        rc = launch_gemm_fp8_tile(up, FP8_GATE_UP, stream);
        if (rc) return rc;
    } else if (wide) {
        up.C = s.codes; up.sc_m = ipad;
        rc = launch_gemm_fp8_wide(up, FP8_GATE_UP, stream);
        if (rc) return rc;
    } else if (a.I > 0) {
        up.C = s.mid; up.sc_m = ipad;
        rc = launch_gemm_fp8(up, FP8_GATE_UP, stream);
        if (rc) return rc;
        tv_quantize_fp8_args q{};
        q.dtype_x = TV_FLOAT32;
        q.block_rows = 1;
        q.M = tk; q.K = a.I;
        q.x = s.mid; q.sx_m = ipad;
        q.q = s.codes; q.sq_m = ipad;
        q.scale = s.mid_scale; q.ss_m = 1; q.ss_k = tk;
        rc = launch_quantize_fp8(q, stream);
        if (rc) return rc;
    }
    down.A = s.codes;
    down.a_scale = s.mid_scale;
    down.C = s.y; down.sc_m = hpad;
    if (tiled && pad_down) {
        rc = pad_fp8_operands(down, FP8_DOWN, pads, stream);
        if (rc) return rc;
    }
    rc = tiled ? launch_gemm_fp8_tile(down, FP8_DOWN, stream) : wide ? launch_gemm_fp8_wide(down, FP8_DOWN, stream) : launch_gemm_fp8(down, FP8_DOWN, stream);
    if (rc) return rc;

    // 2048 columns a workgroup, 512 where those would not fill the CUs.
    const unsigned threads = a.T * ((a.H + 2047) / 2048) >= 4 * device_cus() ? 256 : 64;
    const int64_t wgs = a.T * ((a.H + threads * 8 - 1) / (threads * 8));
    const dim3 grid((unsigned)(wgs < kMaxGrid ? wgs : kMaxGrid));
    auto sum = [&](auto zero) {
        using T = decltype(zero);
        if (tiled)
            hipLaunchKernelGGL((experts_sum_kernel<T, _Float16>), grid, dim3(threads), 0, stream, static_cast<const _Float16*>(s.y), hpad, s.row_scale,
                               ld, s.slot_row, a.T, a.H, a.k, static_cast<T*>(a.C), a.sc_m);
        else
            hipLaunchKernelGGL((experts_sum_kernel<T, float>), grid, dim3(threads), 0, stream, static_cast<const float*>(s.y), hpad, nullptr, 0,
                               s.slot_row, a.T, a.H, a.k, static_cast<T*>(a.C), a.sc_m);
        return (int)hipGetLastError();
    };
    switch (a.dtype_c) {
        case TV_BFLOAT16: return sum((__bf16)0.0f);
        case TV_FLOAT16: return sum((_Float16)0.0f);
        default: return sum(0.0f);
    }
}

// Calls of very many slots run in parts of whole tokens: the rows' offsets stay within 31 bits, and the workspace does
// not grow with the batch.
constexpr int64_t kPartSlots = (int64_t)1 << 19;

int launch_experts_fp8(const tv_experts_fp8_args& a, hipStream_t stream) {
    const int64_t span = a.sa_m > 4 * a.sas_m ? a.sa_m : 4 * a.sas_m; // bytes from token to token
    const int64_t room = (((int64_t)1 << 31) - ((int64_t)1 << 21)) / (span > 0 ? span : 1);
    const int64_t most = kPartSlots / a.k, part = room < 1 ? 1 : room < most ? room : most;
    for (int64_t t = 0; t < a.T; t += part) {
        tv_experts_fp8_args p = a;
        p.T = a.T - t < part ? a.T - t : part;
        p.A = static_cast<const uint8_t*>(a.A) + t * a.sa_m;
        p.a_scale = a.a_scale + t * a.sas_m;
        p.ids = a.ids + t * a.k;
        p.weights = a.weights + t * a.k;
        p.C = static_cast<char*>(a.C) + t * a.sc_m * (int64_t)dtype_size(a.dtype_c);
        const int rc = run_experts(p, stream);
        if (rc) return rc;
    }
    return 0;
}

} // namespace tvk
