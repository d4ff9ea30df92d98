// Quantisation to e4m3 blocks, and the root-mean-square norm with the residual's addition that quantises
// its result: both are one pass over their rows and bound by HBM.
#include "fp8_common.h"

namespace tvk {

// 1 x 128 blocks.  16 lanes hold one block, 8 elements each (a 16-bit lane loads 16 bytes), so the
// largest magnitude is four DPP steps inside a row of 16 lanes and nothing is shared between waves.  bf16 [8192,4096] 20 us, 5.0 TB/s;
// [777,1003] in fp32 3 us.
template <typename T, bool SHORT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(tv_quantize_fp8_args a, int64_t nblocks, int64_t kb) {
    for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < nblocks; i += (int64_t)gridDim.x * 16) {
        int64_t m, b;
        if (nblocks < ((int64_t)1 << 32)) { // uniform: 32-bit division where it suffices
            m = (uint32_t)i / (uint32_t)kb;
            b = (uint32_t)i - (uint32_t)m * (uint32_t)kb;
        } else {
            m = i / kb;
            b = i - m * kb;
        }
        const int64_t k = b * TV_FP8_BLOCK + (threadIdx.x & 15) * 8, left = a.K - k;
        float v[8];
        Eight<T, SHORT> x;
        x.load(static_cast<const T*>(a.x) + m * a.sx_m, k, a.K);
        x.get(k, a.K, v);
        unsigned mx = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = umax(mx, abs_bits(v[j]));
        const Fp8Block f = fp8_block(row16_max(mx));
        store_codes8(static_cast<uint8_t*>(a.q) + m * a.sq_m + k, left, v, f);
        if ((threadIdx.x & 15) == 0) a.scale[m * a.ss_m + b * a.ss_k] = f.scale;
    }
}

// 128 x 128 blocks, one workgroup each: 16 lanes take 8 elements of a row, 512 threads 32 rows, in 4 steps whose values
// stay in registers between the search for the largest magnitude and the conversion.  Bound by HBM: bf16 [11008,4096]
// 22-25 us, 5.4 TB/s or more, part of x in the caches; 28 with inputs that are not (before the vector loads of the rows' ends: 29.1;
// with 256 threads and 8 steps 32.8; four blocks side by side in a workgroup, whole rows of 1 KB but
// half the waves on a CU, 34.6).
template <typename T, bool SHORT>
__global__ __launch_bounds__(512) void quantize_tiles_kernel(tv_quantize_fp8_args a, int64_t kb, int64_t first) {
    __shared__ unsigned part[8];
    const int64_t at = first + blockIdx.x, mb = at / kb, b = at - mb * kb;
    const int64_t k = b * TV_FP8_BLOCK + (threadIdx.x & 15) * 8, left = a.K - k;
    const int64_t m0 = mb * TV_FP8_BLOCK + (threadIdx.x >> 4);
    Eight<T, SHORT> x[4];
    float v[4][8];
    unsigned mx = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + 32 * i;
        x[i].load(static_cast<const T*>(a.x) + (m < a.M ? m : a.M - 1) * a.sx_m, k, a.K); // rows past the end repeat the last one
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i].get(k, a.K, v[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = umax(mx, abs_bits(v[i][j]));
    mx = row16_max(mx);
    mx = umax(mx, (unsigned)__shfl_xor((int)mx, 16));
    mx = umax(mx, (unsigned)__shfl_xor((int)mx, 32));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = umax(mx, part[w]);
    const Fp8Block f = fp8_block(mx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + 32 * i;
        if (m < a.M) store_codes8(static_cast<uint8_t*>(a.q) + m * a.sq_m + k, left, v[i], f);
    }
    if (threadIdx.x == 0) a.scale[mb * a.ss_m + b * a.ss_k] = f.scale;
}

template <typename T, bool SHORT> static int quantize(const tv_quantize_fp8_args& a, hipStream_t stream) {
    const int64_t kb = (a.K + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK;
    if (a.block_rows == 1) {
        const int64_t n = a.M * kb, wgs = (n + 15) / 16;
        hipLaunchKernelGGL((quantize_rows_kernel<T, SHORT>), dim3((unsigned)(wgs < kMaxGrid ? wgs : kMaxGrid)), dim3(256), 0, stream, a, n, kb);
    } else {
        const int64_t n = (a.M + TV_FP8_BLOCK - 1) / TV_FP8_BLOCK * kb;
        for (int64_t first = 0; first < n; first += kMaxGrid) {
            hipLaunchKernelGGL((quantize_tiles_kernel<T, SHORT>), dim3((unsigned)(n - first < kMaxGrid ? n - first : kMaxGrid)), dim3(512), 0, stream, a, kb, first);
            const int rc = hipGetLastError();
            if (rc) return rc;
        }
        return 0;
    }
    return hipGetLastError();
}

int launch_quantize_fp8(const tv_quantize_fp8_args& a, hipStream_t stream) {
    switch (a.dtype_x) {
        case TV_BFLOAT16: return a.K < 8 ? quantize<__bf16, true>(a, stream) : quantize<__bf16, false>(a, stream);
        case TV_FLOAT16: return a.K < 8 ? quantize<_Float16, true>(a, stream) : quantize<_Float16, false>(a, stream);
        default: return a.K < 8 ? quantize<float, true>(a, stream) : quantize<float, false>(a, stream);
    }
}

// y = v * rsqrt(mean(v^2) + eps) * weight with v = x + residual, one workgroup per row.  A thread holds CH chunks of 8
// elements; chunk c of step i is thread c's, so 16 lanes hold a block of 128 and the row is read once:
// v stays in registers over the sum of squares.  CH = 0: rows too long for the registers of a workgroup;
// they are read a second time.  8192 rows of 4096 in bf16 with residual and normed rows (303 MB): 55-58 us,
// 5.4 TB/s (rows of 4095: 74); one row 3 us.
template <typename T, typename W, int BT, int CH, bool SHORT = false>
__global__ __launch_bounds__(BT) void rms_norm_fp8_kernel(tv_rms_norm_fp8_args a) {
    constexpr int NW = BT / 64, STEP = BT * 8;
    __shared__ float part[NW];
    const int tid = threadIdx.x;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + t * a.sx;
        const T* r = a.residual ? static_cast<const T*>(a.residual) + t * a.sr : nullptr;
        const W* w = static_cast<const W*>(a.weight);
        constexpr int N = CH ? CH : 1;
        auto read = [&](int64_t k0, float (&v)[N][8]) {
            constexpr int G = N < 2 ? N : 2; // chunks on their way at once: four would not fit the registers
#pragma unroll
            for (int i0 = 0; i0 < N; i0 += G) {
                Eight<T, SHORT> ex[G], er[G];
#pragma unroll
                for (int i = 0; i < G; ++i) ex[i].load(x, k0 + (int64_t)(i0 + i) * STEP, a.H);
                if (r)
#pragma unroll
                    for (int i = 0; i < G; ++i) er[i].load(r, k0 + (int64_t)(i0 + i) * STEP, a.H);
#pragma unroll
                for (int i = 0; i < G; ++i) ex[i].get(k0 + (int64_t)(i0 + i) * STEP, a.H, v[i0 + i]);
                if (r)
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        float u[8];
                        er[i].get(k0 + (int64_t)(i0 + i) * STEP, a.H, u);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[i0 + i][j] += u[j];
                    }
            }
        };
        auto write = [&](int64_t k, float (&v)[8], float rstd) {
            const int64_t left = a.H - k;
            if (a.residual_out) store8(static_cast<T*>(a.residual_out) + t * a.sro + k, left, v);
            float g[8];
            Eight<W, SHORT> weight;
            weight.load(w, k, a.H);
            weight.get(k, a.H, g);
            unsigned mx = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = v[j] * rstd * g[j];
                mx = umax(mx, abs_bits(v[j]));
            }
            const Fp8Block f = fp8_block(row16_max(mx));
            if (a.normed) store8(static_cast<T*>(a.normed) + t * a.sn + k, left, v);
            store_codes8(static_cast<uint8_t*>(a.q) + t * a.sq + k, left, v, f);
            if ((tid & 15) == 0 && left > 0) a.scale[t * a.ss_m + k / TV_FP8_BLOCK * a.ss_k] = f.scale;
        };
        float sum = 0.0f;
        float v[N][8];
        if constexpr (CH > 0) {
            read(tid * 8, v);
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
        } else {
            for (int64_t k = tid * 8; k < a.H; k += STEP) {
                read(k, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += v[0][j] * v[0][j];
            }
        }
        sum = wave_sum(sum);
        if constexpr (NW > 1) {
            __syncthreads(); // the previous row's sums are read
            if ((tid & 63) == 0) part[tid >> 6] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NW; ++i) sum += part[i];
        }
        const float rstd = 1.0f / sqrtf(sum / (float)a.H + a.eps);
        if constexpr (CH > 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int64_t k = (int64_t)i * STEP + tid * 8;
                // The 16 lanes of a block take part together: a whole block past the row is skipped.
                if (k / TV_FP8_BLOCK * TV_FP8_BLOCK < a.H) write(k, v[i], rstd);
            }
        } else {
            for (int64_t k = tid * 8; k / TV_FP8_BLOCK * TV_FP8_BLOCK < a.H; k += STEP) {
                read(k, v);
                write(k, v[0], rstd);
            }
        }
    }
}

template <typename T, typename W> static int rms_norm(const tv_rms_norm_fp8_args& a, hipStream_t stream) {
    const unsigned grid = (unsigned)(a.T < kMaxGrid ? a.T : kMaxGrid);
    auto run = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, stream, a);
        return (int)hipGetLastError();
    };
    // us in bf16 with residual, without normed rows, 1 row and 8192 rows, against half as many threads with twice the chunks (H 512: four times as many
    // threads): H 512 2.8, 6.7 (2.8, 12.8); 2048 2.9, 21.3 (3.6, 22.3); 4096 3.2, 40 (3.8, 40); 8192 4.0, 95 (5.6, 100; 1024
    // threads 4.0, 97); 16384 5.0, 207 (6.2, 243 with 4 chunks).
    if (a.H < 8) return run(rms_norm_fp8_kernel<T, W, 64, 1, true>, 64);
    if (a.H <= 512) return run(rms_norm_fp8_kernel<T, W, 64, 1>, 64);
    if (a.H <= 2048) return run(rms_norm_fp8_kernel<T, W, 256, 1>, 256);
    if (a.H <= 4096) return run(rms_norm_fp8_kernel<T, W, 512, 1>, 512);
    if (a.H <= 8192) return run(rms_norm_fp8_kernel<T, W, 512, 2>, 512);
    if (a.H <= 16384) return run(rms_norm_fp8_kernel<T, W, 1024, 2>, 1024);
    if (a.H <= 32768) return run(rms_norm_fp8_kernel<T, W, 1024, 4>, 1024);
    return run(rms_norm_fp8_kernel<T, W, 1024, 0>, 1024);
}

int launch_rms_norm_fp8(const tv_rms_norm_fp8_args& a, hipStream_t stream) {
    const bool wide = a.dtype_w == TV_FLOAT32;
    switch (a.dtype_x) {
        case TV_BFLOAT16: return wide ? rms_norm<__bf16, float>(a, stream) : rms_norm<__bf16, __bf16>(a, stream);
        case TV_FLOAT16: return wide ? rms_norm<_Float16, float>(a, stream) : rms_norm<_Float16, _Float16>(a, stream);
        default: return rms_norm<float, float>(a, stream);
    }
}

} // namespace tvk
