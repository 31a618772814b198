// Rows in 8 bits with a scale each, and their product with 8-bit weights that
// have a scale for each output channel (sm_100a).
//
//   quantise  s = max(max|x| / 127, 2^-126), q = x / s to the nearest integer
//   product   y[t][n] = x_scale[t] w_scale[n] sum_k x[t][k] w[n][k] + bias[n]
//
// The integer sums are exact (int32; |x w| <= 2^14 and at most 2^17 - 16
// terms), so that the order of a sum, the tile and the kernel that computes it
// do not show in the result: y has the three roundings of float(sum), of its
// product with x_scale and of that with w_scale (and bias), and the one to bf16.
#pragma once

#include "phonon_attention.cuh"
#include "phonon_gemm.cuh"
#include "phonon_kv8_prompt.cuh"

namespace phonon {

// ----------------------------------------------------------------- quantise
struct I8QuantParams {
    const void* x;
    int8_t* q;
    float* scales;
    long long x_stride, q_stride;  // elements
    int32_t* status;               // [rows] or null
    int rows, cols;
};

// The nearest integer to x / s, ties to even: the nearest to x * (1 / s) is
// that but next to a border, and x - q s is exact (of both operands' last bits
// and at most a step large), so that it says on which side x lies.
__device__ __forceinline__ float i8_fix(float q, float x, float s) {
    const float rest = fmaf(-q, s, x), twice = 2.0f * fabsf(rest);  // (half the smallest scales is not a float)
    const bool odd = static_cast<int>(q) & 1;
    if (twice > s || (twice == s && odd)) q += rest > 0.0f ? 1.0f : -1.0f;
    return q;
}

// kThreads threads a row, kUnits units of 8 elements a thread in registers; a
// row of more is read twice. Bound by the bytes.
template <bool kBf16, int kThreads, int kUnits>
__global__ void __launch_bounds__(256) i8_quantize_kernel(I8QuantParams p) {
    constexpr int kRows = 256 / kThreads, kWarps = kThreads / 32;
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    __shared__ uint32_t s_top[8];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % kThreads, warp = threadIdx.x >> 5;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / kThreads;
    const bool there = row < p.rows;
    const int units = there ? p.cols / 8 : 0;
    const size_t in = static_cast<size_t>(row) * p.x_stride;
    float4 v[kUnits][2];
    uint32_t top = 0;  // the largest magnitude's bits; not finite: 0x7f800000 or more
    auto look = [&](float4 a) {
        top = max(top, max(max(__float_as_uint(a.x) & 0x7fffffffu, __float_as_uint(a.y) & 0x7fffffffu),
                           max(__float_as_uint(a.z) & 0x7fffffffu, __float_as_uint(a.w) & 0x7fffffffu)));
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            v[u][h] = u * kThreads + t < units ? load_row4<kBf16>(p.x, in + (u * kThreads + t) * 8 + 4 * h)
                                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) look(v[u][0]), look(v[u][1]);
    for (int u = kUnits * kThreads + t; u < units; u += kThreads) {
        look(load_row4<kBf16>(p.x, in + u * 8ll));
        look(load_row4<kBf16>(p.x, in + u * 8ll + 4));
    }
    top = __reduce_max_sync(kFull, top);
    if constexpr (kWarps > 1) {
        if ((threadIdx.x & 31) == 0) s_top[warp] = top;
        __syncthreads();
        const int first = warp / kWarps * kWarps;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = max(top, s_top[first + w]);
    }
    if (!there) return;
    const bool bad = top >= 0x7f800000u;
    const float s = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 0x1p-126f), inverse = bad ? 0.0f : __frcp_rn(s);
    if (t == 0) {
        p.scales[row] = bad ? __int_as_float(0x7fc00000) : s;
        if (bad) flag_nonfinite(p.status, static_cast<int>(row));
    }
    int8_t* out = p.q + static_cast<size_t>(row) * p.q_stride;
    auto put = [&](const float4 (&x)[2], int u) {
        float q[8], far = 0.0f;
        const float* f = &x[0].x;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float e = bad ? 0.0f : f[k];
            q[k] = fmaf(e, inverse, kRound) - kRound;
            far = fmaxf(far, fabsf(fmaf(-q[k], s, e)));
        }
        if (!bad && 2.0f * far >= s) {
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = i8_fix(q[k], f[k], s);
        }
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(q[k] + kRound);  // the low byte is the integer's
        *reinterpret_cast<uint2*>(out + u * 8ll) = make_uint2(kv8_pack(w[0], w[1], w[2], w[3]), kv8_pack(w[4], w[5], w[6], w[7]));
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
        if (u * kThreads + t < units) put(v[u], u * kThreads + t);
    for (int u = kUnits * kThreads + t; u < units; u += kThreads) {
        const float4 x[2] = {load_row4<kBf16>(p.x, in + u * 8ll), load_row4<kBf16>(p.x, in + u * 8ll + 4)};
        put(x, u);
    }
}

// ------------------------------------------------------------------ product
struct I8Params {
    const int8_t* x;  // [rows][depth]
    const int8_t* w;  // [channels][depth]
    const float* x_scales;
    const float* w_scales;
    const float* bias;  // [channels] or null
    void* y;
    long long x_stride, w_stride, y_stride;
    int32_t* status;  // [rows] or null
    int rows, channels, depth;
    int tiles_m, tiles_n;  // of the tiled kernel
};

__device__ __forceinline__ float i8_value(int sum, float x_scale, float w_scale, float bias) {
    return fmaf(static_cast<float>(sum) * x_scale, w_scale, bias);
}

template <bool kBf16>
__device__ __forceinline__ bool i8_store(void* y, size_t at, float v) {  // whether it is finite as it is held
    if constexpr (kBf16) {
        const __nv_bfloat16 b = __float2bfloat16(v);
        static_cast<__nv_bfloat16*>(y)[at] = b;
        return isfinite(__bfloat162float(b));
    } else {
        static_cast<float*>(y)[at] = v;
        return isfinite(v);
    }
}

// Few rows (a decode step): bound by the weights' bytes. A CTA has 16 channels,
// its warps share the depth and meet in shared memory. The weights are the A
// operand as they lie: lane 4g + t takes 16 bytes of channels g and g + 8 at
// 64c + 16t, whose words count as the depths that the fragments' order asks
// for, in the rows' operand alike, so that nothing is exchanged.
constexpr int kI8Warps = 8, kI8Ahead = 8;

template <int NT, bool kBf16>
__global__ void __launch_bounds__(32 * kI8Warps) i8_rows_kernel(I8Params p) {
    __shared__ int s_sum[kI8Warps][16][8 * NT + 1];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16;
    const int chunks = (p.depth + 63) / 64, per = (chunks + kI8Warps - 1) / kI8Warps;
    const int first = min(chunks, warp * per), last = min(chunks, first + per);
    const int8_t* w0 = p.w + static_cast<size_t>(min(n0 + g, p.channels - 1)) * p.w_stride + 16 * t;
    const int8_t* w1 = p.w + static_cast<size_t>(min(n0 + g + 8, p.channels - 1)) * p.w_stride + 16 * t;
    const int8_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = p.x + static_cast<size_t>(min(8 * n + g, p.rows - 1)) * p.x_stride + 16 * t;
    int sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0;
    constexpr int kAhead = NT > 2 ? kI8Ahead / 2 : kI8Ahead;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c0 = first; c0 < last; c0 += kAhead) {
        uint4 a[kAhead][2], b[kAhead][NT];
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
            const int k = (c0 + c) * 64;
            const bool in = c0 + c < last && k + 16 * t < p.depth;
            a[c][0] = in ? *reinterpret_cast<const uint4*>(w0 + k) : zero;
            a[c][1] = in ? *reinterpret_cast<const uint4*>(w1 + k) : zero;
#pragma unroll
            for (int n = 0; n < NT; ++n) b[c][n] = in ? *reinterpret_cast<const uint4*>(x[n] + k) : zero;
        }
#pragma unroll
        for (int c = 0; c < kAhead; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                imma_s8_s8(sum[n], sum[n], a[c][0].x, a[c][1].x, a[c][0].y, a[c][1].y, b[c][n].x, b[c][n].y);
                imma_s8_s8(sum[n], sum[n], a[c][0].z, a[c][1].z, a[c][0].w, a[c][1].w, b[c][n].z, b[c][n].w);
            }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) s_sum[warp][g + 8 * (k >> 1)][8 * n + 2 * t + (k & 1)] = sum[n][k];
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * 8 * NT; at += 32 * kI8Warps) {
        const int c = at & 15, row = at >> 4, n = n0 + c;
        if (row >= p.rows || n >= p.channels) continue;
        int total = 0;
#pragma unroll
        for (int k = 0; k < kI8Warps; ++k) total += s_sum[k][c][row];
        const float v = i8_value(total, p.x_scales[row], p.w_scales[n], p.bias ? p.bias[n] : 0.0f);
        if (!i8_store<kBf16>(p.y, static_cast<size_t>(row) * p.y_stride + n, v)) flag_nonfinite(p.status, row);
    }
}

// A bounded wait, whatever has failed.
__device__ __forceinline__ void mbar_settle(uint32_t bar, uint32_t parity) {
    for (const long long since = clock64(); !mbar_test(bar, parity) && clock64() - since < kWaitBudgetCycles;) __nanosleep(20);
}

// Many rows: tiles of 128 rows x kN channels on the tcgen05 tensor cores, one
// CTA an SM that takes tiles in turn. Warp 0 brings 128 bytes of depth a stage
// by TMA, warp 1 issues the products into one of two accumulators in TMEM, and
// warps 2-5 take the other one out, a row a thread.
constexpr int kI8Threads = 192;

template <int kN>
__host__ __device__ constexpr int i8_stages() { return kN == 256 ? 4 : kN == 128 ? 6 : 8; }

template <int kN>
__host__ __device__ constexpr int i8_smem() { return 1024 + i8_stages<kN>() * (128 + kN) * 128; }

template <int kN, bool kBf16>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_product_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, I8Params p) {
    constexpr int kStages = i8_stages<kN>(), kStageBytes = (128 + kN) * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * kStages + 5];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(16) float s_scale[2][kN], s_bias[2][kN];
    const uint32_t stages = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = smem_addr(s_bars), empty = full + 8 * kStages, done = empty + 8 * kStages, drained = done + 16, idle = drained + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(done + 8 * a, 1);
            mbar_init(drained + 8 * a, 4);
        }
        mbar_init(idle, 1);
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(2 * kN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    const int nk = (p.depth + 127) / 128, tiles = p.tiles_m * p.tiles_n;
    // Tiles in bands of kBand row tiles, so that the CTAs at work share rows and weights in the L2.
    constexpr int kBand = 16;
    auto place = [&](int tile, int& m, int& n) {
        const int band = tile / (kBand * p.tiles_n), in = tile - band * kBand * p.tiles_n;
        const int high = min(kBand, p.tiles_m - band * kBand);
        n = in / high;
        m = band * kBand + in - n * high;
    };
    pdl_wait();
    pdl_trigger();
    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
            int m, n;
            place(tile, m, n);
            for (int k = 0; k < nk; ++k, ++it) {
                const int s = it % kStages;
                if (it >= kStages && !(ok = mbar_wait(empty + 8 * s, (it / kStages - 1) & 1, nullptr, &s_failed))) break;
                mbar_expect_tx(full + 8 * s, kStageBytes);
                tma_load_2d(stages + s * kStageBytes, &tm_x, k * 128, m * 128, full + 8 * s);
                tma_load_2d(stages + s * kStageBytes + 128 * 128, &tm_w, k * 128, n * kN, full + 8 * s);
            }
        }
        if (!ok)  // a wait ran out: no copy is on its way when the CTA gives its memory back
            for (int j = max(0, it - kStages); j < it; ++j) mbar_settle(full + 8 * (j % kStages), (j / kStages) & 1);
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = umma_idesc_i8(128, kN);
        int it = 0, turn = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++turn) {
            const int a = turn & 1;
            if (turn >= 2 && !(ok = mbar_wait(drained + 8 * a, (turn / 2 - 1) & 1, nullptr, &s_failed))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int k = 0; k < nk; ++k, ++it) {
                const int s = it % kStages;
                if (!(ok = mbar_wait(full + 8 * s, (it / kStages) & 1, nullptr, &s_failed))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = stages + s * kStageBytes;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_i8(tmem + a * kN, umma_desc_sw128(at + kk * 32), umma_desc_sw128(at + 128 * 128 + kk * 32), idesc, (k | kk) != 0);
                umma_commit(empty + 8 * s);
            }
            if (ok) umma_commit(done + 8 * a);
        }
        umma_commit(idle);  // nor is a product
        mbar_settle(idle, 0);
    } else if (warp >= 2) {
        const int quarter = warp & 3, thread = (warp - 2) * 32 + lane;
        int turn = 0;
        const bool wide = p.y_stride % (kBf16 ? 8 : 4) == 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
            int m, n;
            place(tile, m, n);
            const int a = turn & 1, n0 = n * kN, row = m * 128 + quarter * 32 + lane;
            for (int c = thread; c < kN; c += 128) {
                s_scale[a][c] = n0 + c < p.channels ? p.w_scales[n0 + c] : 0.0f;
                s_bias[a][c] = p.bias && n0 + c < p.channels ? p.bias[n0 + c] : 0.0f;
            }
            float xs = row < p.rows ? p.x_scales[row] : 0.0f;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            mbar_wait(done + 8 * a, (turn / 2) & 1, nullptr, &s_failed);
            __syncwarp();
            const bool failed = *static_cast<volatile int*>(&s_failed);
            if (failed) xs = __int_as_float(0x7fc00000);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const size_t out = static_cast<size_t>(row) * p.y_stride + n0;
            float finite = 0.0f;
#pragma unroll 1
            for (int c = 0; c < kN; c += 32) {
                uint32_t r[32];
                tmem_load32(tmem + a * kN + c + (static_cast<uint32_t>(quarter * 32) << 16), r);
                if (c + 32 >= kN) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(drained + 8 * a);
                }
                if (row >= p.rows || n0 + c >= p.channels) continue;
                float v[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    v[k] = i8_value(static_cast<int>(r[k]), xs, s_scale[a][c + k], s_bias[a][c + k]);
                    if constexpr (kBf16) v[k] = __bfloat162float(__float2bfloat16(v[k]));
                    if (n0 + c + k < p.channels) finite = fmaf(v[k], 0.0f, finite);
                }
                if (wide && n0 + c + 32 <= p.channels) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) store_row4<kBf16>(p.y, out + c + k, make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (n0 + c + k < p.channels) i8_store<kBf16>(p.y, out + c + k, v[k]);
                }
            }
            if (row < p.rows && finite != 0.0f) flag_nonfinite(p.status, row);
            if (failed && row < p.rows && p.status) atomicMax(p.status + row, kStatusDevice);
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * kN) : "memory");
    }
}

}  // namespace phonon
