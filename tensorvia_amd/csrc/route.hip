// Routing: the k experts of each token.
//
// LPT lanes (16 or 64) work on one token; a lane holds EPL consecutive experts, so a token's logits are read once
// and everything stays in registers.  What a token's lanes share goes through lane permutations that are moves of
// the vector ALU (DPP inside 16 lanes, permlane swaps across), none through LDS: with 64 lanes a token and
// LDS permutations 16384 tokens of 64 experts took 25.8 us, bound by LDS (130 permutations a token); now 5.9, bound by the vector
// ALU.  64 tokens of 256 experts in groups 5.6 us: the dependent steps of one token's choice.
//
// A round of the choice: the largest value (as order-preserving bits, one maximum), then the lowest index that
// has it (one minimum).  Scores wait in LDS for the k indices.
//
// The softmax's denominator is summed in 64 bits and rounded to fp32 once.  Up to 1024 terms in [0, 1], the largest 1: in any order
// the 64-bit sum is off by at most 1024 * 2^-53 = 2^-43 of itself, so two orders (16 lanes or 64 a token) give scores that differ only
// where the sum lies that close to the middle between two fp32 numbers: one sum in 2^18 at the very most.
#include "fp8_common.h"

namespace tvk {

__device__ inline unsigned order_bits(float x) { // increasing in x; 0 is below every number's
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f); // -0 counts as 0
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

// Step D of a butterfly over up to 64 lanes: each lane gets the value of a lane in the other half of its 2 D lanes.
// (From 4 lanes on the halves hold equal values in all their lanes, so any lane of the other half will do.)
template <int D> __device__ inline unsigned other(unsigned x) {
    constexpr int ctrl = D == 1 ? 0xB1 /* quad_perm 1,0,3,2 */ : D == 2 ? 0x4E /* 2,3,0,1 */ : D == 4 ? 0x141 /* half row mirror */ : 0x140 /* row mirror */;
    if constexpr (D <= 8) return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);
    // The swaps leave one half's values in both halves of one result, and the other half's in the other.
    const auto p = [&] {
        if constexpr (D == 16) return __builtin_amdgcn_permlane16_swap(x, x, false, false);
        else return __builtin_amdgcn_permlane32_swap(x, x, false, false);
    }();
    return (threadIdx.x & D) ? p[0] : p[1];
}
template <int D> __device__ inline double other(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)other<D>((unsigned)(u >> 32)) << 32 | other<D>((unsigned)u));
}
template <int D> __device__ inline float other(float x) { return __builtin_bit_cast(float, other<D>(__builtin_bit_cast(unsigned, x))); }
// op over the first N lanes' butterfly steps (N a power of two up to 64), the result in all of them.
template <int N, typename T, typename F> __device__ inline T butterfly(T x, const F& op) {
    if constexpr (N >= 2) x = op(x, other<1>(x));
    if constexpr (N >= 4) x = op(x, other<2>(x));
    if constexpr (N >= 8) x = op(x, other<4>(x));
    if constexpr (N >= 16) x = op(x, other<8>(x));
    if constexpr (N >= 32) x = op(x, other<16>(x));
    if constexpr (N >= 64) x = op(x, other<32>(x));
    return x;
}
__device__ inline unsigned umin(unsigned a, unsigned b) { return a < b ? a : b; }

constexpr int kRouteThreads = 256;
__device__ inline int padded(int e) { return e + (e >> 5); } // groups of a multiple of 32 experts on distinct LDS banks

template <typename T, int LPT, int EPL>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(tv_route_args a) {
    constexpr int TPB = kRouteThreads / LPT; // tokens of a workgroup
    __shared__ float scores[TPB][LPT * EPL];
    __shared__ float values[TPB][LPT * EPL * 33 / 32 + 1]; // groups only, padded()
    const int lane = threadIdx.x & (LPT - 1), slot = threadIdx.x / LPT;
    const int e0 = lane * EPL;
    const float inf = __builtin_inff();
    // All lanes of a wave stay in step: tokens past the end repeat the last one and are not stored.
    for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < a.T; t0 += (int64_t)gridDim.x * TPB) {
        const bool in = t0 + slot < a.T;
        const int64_t t = in ? t0 + slot : a.T - 1;
        const T* row = static_cast<const T*>(a.logits) + t * a.sl + e0;
        float s[EPL]; // logits, then scores
        unsigned live = 0; // bit i: expert e0 + i may be chosen
        if (e0 + EPL <= a.E) {
            T v[EPL];
            __builtin_memcpy(v, row, sizeof(v));
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = (float)v[i];
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = e0 + i < a.E ? (float)row[i] : -inf;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const bool ok = s[i] > -inf; // false for NaN
            live |= ok ? 1u << i : 0;
            s[i] = ok ? fminf(s[i], 3.402823466e38f) : -inf;
        }
        if (a.scoring == TV_SCORE_SOFTMAX) {
            float top = s[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) top = fmaxf(top, s[i]);
            const unsigned m = butterfly<LPT>(order_bits(top), umax);
            top = __builtin_bit_cast(float, m & 0x80000000u ? m ^ 0x80000000u : ~m);
            top = top == -inf ? 0.0f : top;
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                s[i] = expf(s[i] - top);
                sum += (double)s[i];
            }
            sum = butterfly<LPT>(sum, [](double x, double y) { return x + y; });
            const float total = sum == 0.0 ? 1.0f : (float)sum;
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = s[i] / total;
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i) s[i] = 1.0f / (1.0f + expf(-s[i]));
        }
        unsigned key[EPL]; // 0: not to be chosen
        float c[EPL];
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            scores[slot][e0 + i] = s[i];
            c[i] = a.bias && e0 + i < a.E ? s[i] + a.bias[e0 + i] : s[i];
            key[i] = (live >> i & 1) && c[i] > -inf ? order_bits(c[i]) : 0;
            if (!key[i]) c[i] = -inf;
        }
        if (a.groups > 1) {
            // A power of two of lanes per group: each takes its share of the group's values from LDS, and they merge their
            // best two.  The best groups are found like the best experts.
            const int per = a.E / a.groups;
            const int lpg = 1 << (31 - __builtin_clz(LPT / a.groups));
            const int g = lane / lpg;
#pragma unroll
            for (int i = 0; i < EPL; ++i) values[slot][padded(e0 + i)] = c[i];
            __builtin_amdgcn_wave_barrier();
            float b0 = -inf, b1 = -inf;
            if (g < a.groups)
                for (int i = lane - g * lpg; i < per; i += lpg) {
                    const float v = values[slot][padded(g * per + i)];
                    b1 = v > b0 ? b0 : (v > b1 ? v : b1);
                    b0 = v > b0 ? v : b0;
                }
            auto merge = [&](float o0, float o1) {
                b1 = fmaxf(fminf(b0, o0), fmaxf(b1, o1));
                b0 = fmaxf(b0, o0);
            };
            if (lpg >= 2) merge(other<1>(b0), other<1>(b1));
            if (lpg >= 4) merge(other<2>(b0), other<2>(b1));
            if (lpg >= 8) merge(other<4>(b0), other<4>(b1));
            if (lpg >= 16) merge(other<8>(b0), other<8>(b1));
            if (lpg >= 32) merge(other<16>(b0), other<16>(b1));
            unsigned gkey = b0 > -inf ? order_bits(a.group_top == 2 && b1 > -inf ? b0 + b1 : b0) : 0;
            uint64_t kept = 0;
            for (int j = 0; j < a.topk_groups; ++j) {
                const unsigned best = butterfly<LPT>(gkey, umax);
                const unsigned which = butterfly<LPT>(best && gkey == best ? (unsigned)g : ~0u, umin);
                if (which < 64) kept |= (uint64_t)1 << which;
                if (which == (unsigned)g) gkey = 0;
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (e0 + i < a.E && !(kept >> ((e0 + i) / per) & 1)) key[i] = 0;
        }
        // Round j leaves its choice in the token's lane j.
        int id = -1;
        for (int j = 0; j < a.k; ++j) {
            unsigned best = key[0];
#pragma unroll
            for (int i = 1; i < EPL; ++i) best = umax(best, key[i]);
            best = butterfly<LPT>(best, umax);
            unsigned e = ~0u;
#pragma unroll
            for (int i = EPL - 1; i >= 0; --i) e = key[i] == best ? e0 + i : e;
            e = best ? e : ~0u;
            e = butterfly<LPT>(e, umin);
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = e == (unsigned)(e0 + i) ? 0 : key[i];
            if (lane == j) id = (int)e;
        }
        __builtin_amdgcn_wave_barrier();
        float w = id >= 0 ? scores[slot][id] : 0.0f;
        if (a.renormalize) w = w / (butterfly<LPT>(w, [](float x, float y) { return x + y; }) + 1e-20f);
        if (in && lane < a.k) {
            a.weights[t * a.k + lane] = w * a.scale;
            a.ids[t * a.k + lane] = id;
        }
        __builtin_amdgcn_wave_barrier(); // the next tokens' scores follow
    }
}

template <typename T, int LPT, int EPL> static int run_route(const tv_route_args& a, hipStream_t stream) {
    const int64_t wgs = (a.T + kRouteThreads / LPT - 1) / (kRouteThreads / LPT);
    hipLaunchKernelGGL((route_kernel<T, LPT, EPL>), dim3((unsigned)(wgs < kMaxGrid ? wgs : kMaxGrid)), dim3(kRouteThreads), 0, stream, a);
    return hipGetLastError();
}

// 16 lanes a token do the lane permutations of four tokens at once; where that leaves CUs idle, or a token needs more lanes
// (k or groups above 16, experts above 16 a lane), it gets the wave.  us, 16 lanes / 64, 64 experts: 1024 tokens 3.9 / 3.7, 2048
// 4.0 / 4.2, 4096 4.0 / 5.5, 16384 6.0 / 13.8; 256 experts: 2048 7.2 / 5.2, 4096 7.3 / 7.4, 8192 9.1 / 11.8.
constexpr int64_t kRouteNarrowTokens = 4096;

template <typename T> static int route(const tv_route_args& a, hipStream_t stream) {
    if (a.T >= kRouteNarrowTokens && a.k <= 16 && a.groups <= 16 && a.E <= 256) {
        if (a.E <= 16) return run_route<T, 16, 1>(a, stream);
        if (a.E <= 64) return run_route<T, 16, 4>(a, stream);
        if (a.E <= 128) return run_route<T, 16, 8>(a, stream);
        return run_route<T, 16, 16>(a, stream);
    }
    if (a.E <= 64) return run_route<T, 64, 1>(a, stream);
    if (a.E <= 128) return run_route<T, 64, 2>(a, stream);
    if (a.E <= 256) return run_route<T, 64, 4>(a, stream);
    if (a.E <= 512) return run_route<T, 64, 8>(a, stream);
    return run_route<T, 64, 16>(a, stream);
}

int launch_route(const tv_route_args& a, hipStream_t stream) {
    switch (a.dtype) {
        case TV_BFLOAT16: return route<__bf16>(a, stream);
        case TV_FLOAT16: return route<_Float16>(a, stream);
        default: return route<float>(a, stream);
    }
}

} // namespace tvk
