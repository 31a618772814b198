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

// fp32 rows: the nearest integer to x / s, ties to even. The nearest to
// x * (1 / s) is that but next to a border, and x - q s is exact (of both
// operands' last bits and at most a step large), so that it says on which side
// x lies.
__device__ __forceinline__ float i8_fix(float q, float x, float s) {
    const float rest = fmaf(-q, s, x), twice = 2.0f * fabsf(rest);  // (half the smallest scales is not a float)
    const bool odd = static_cast<int>(q) & 1;
    if (twice > s || (twice == s && odd)) q += rest > 0.0f ? 1.0f : -1.0f;
    return q;
}

// Eight elements of a row as they lie.
template <bool kBf16>
struct I8Unit {
    uint4 w[kBf16 ? 1 : 2];
    __device__ __forceinline__ void load(const void* x, size_t at) {
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + at * (kBf16 ? 2 : 4));
        w[0] = from[0];
        if constexpr (!kBf16) w[1] = from[1];
    }
    __device__ __forceinline__ void zero() {
        w[0] = make_uint4(0, 0, 0, 0);
        if constexpr (!kBf16) w[1] = w[0];
    }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& v = w[i / 4];
        return i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w;
    }
    __device__ __forceinline__ float element(int k) const {
        if constexpr (kBf16) return __uint_as_float(k % 2 ? word(k / 2) & 0xffff0000u : word(k / 2) << 16);
        else return __uint_as_float(word(k));
    }
    // The largest magnitude's bits so far (of bf16 in both halves).
    __device__ __forceinline__ uint32_t top(uint32_t most) const {
#pragma unroll
        for (int i = 0; i < (kBf16 ? 4 : 8); ++i)
            most = kBf16 ? __vmaxu2(most, word(i) & 0x7fff7fffu) : max(most, word(i) & 0x7fffffffu);
        return most;
    }
};

// CTAs an SM: as many as registers hold without spills (rows of 256 bf16: 18.1
// us for 100000, with 4 CTAs an SM 20.6; 20000 of 512: 6.7, 9.8).
template <bool kBf16, int kUnits>
__host__ __device__ constexpr int i8_quantize_ctas() {
    return kBf16 ? kUnits == 1 ? 8 : kUnits == 2 ? 6 : 4 : kUnits == 1 ? 5 : kUnits == 2 ? 4 : 2;
}

// kThreads threads a row, kUnits units of 8 elements a thread in registers, as
// they lie, the next row's on their way meanwhile; a row of more is read twice.
// Bound by the bytes: 8192 x 4096 bf16 in 16.7 us (6.0 TB/s, 92 % of a plain
// copy's rate), fp32 in 26.2 (6.4). Short rows by their first loads: 64 x 512
// fp32 in 1.7.
template <bool kBf16, int kThreads, int kUnits>
__global__ void __launch_bounds__(256, i8_quantize_ctas<kBf16, kUnits>()) i8_quantize_kernel(I8QuantParams p) {
    constexpr int kRows = 256 / kThreads, kWarps = kThreads / 32;
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    __shared__ uint32_t s_top[2][8];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % kThreads, warp = threadIdx.x >> 5, units = p.cols / 8;
    const int step = static_cast<int>(gridDim.x) * kRows;
    I8Unit<kBf16> v[kUnits], next[kUnits];
    const auto load = [&](I8Unit<kBf16> (&x)[kUnits], long long row) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (row < p.rows && u * kThreads + t < units) x[u].load(p.x, static_cast<size_t>(row) * p.x_stride + (u * kThreads + t) * 8ll);
            else x[u].zero();
        }
    };
    const int own = threadIdx.x / kThreads;
    load(next, blockIdx.x * static_cast<long long>(kRows) + own);
    int parity = 0;
    for (long long base = blockIdx.x * static_cast<long long>(kRows); base < p.rows; base += step, parity ^= 1) {
        const long long row = base + own;
        const bool there = row < p.rows;
        const size_t in = static_cast<size_t>(row) * p.x_stride;
        uint32_t top = 0;  // the largest magnitude's bits; not finite: an exponent of ones
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            v[u] = next[u];
            top = v[u].top(top);
        }
        load(next, row + step);
        for (int u = kUnits * kThreads + t; there && u < units; u += kThreads) {
            I8Unit<kBf16> x;
            x.load(p.x, in + u * 8ll);
            top = x.top(top);
        }
        if constexpr (kBf16) top = max(top & 0xffff0000u, top << 16);
        top = __reduce_max_sync(kFull, top);
        if constexpr (kWarps > 1) {
            if ((threadIdx.x & 31) == 0) s_top[parity][warp] = top;
            __syncthreads();
            const int first = warp / kWarps * kWarps;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = max(top, s_top[parity][first + w]);
        }
        if (!there) continue;
        const bool bad = top >= 0x7f800000u;
        const float s = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 0x1p-126f);
        float inverse = __frcp_rn(s);
        // bf16: x / s is k + 1/2 but for the rounding of s, or further from it than a few roundings (both have 8 bits
        // but for the 127). So the product with a reciprocal that errs to the side of x / s rounds as x / s does:
        // a step down where s is above top / 127, one up below it.
        if constexpr (kBf16) {
            const float over = fmaf(s, 127.0f, -__uint_as_float(top));
            if (s > 0x1p-126f) inverse = __int_as_float(__float_as_int(inverse) - (over > 0.0f) + (over < 0.0f));
        }
        if (t == 0) {
            p.scales[row] = bad ? __int_as_float(0x7fc00000) : s;
            if (bad) flag_nonfinite(p.status, static_cast<int>(row));
        }
        int8_t* out = p.q + static_cast<size_t>(row) * p.q_stride;
        auto put = [&](const I8Unit<kBf16>& x, int u) {
            uint32_t w[8];  // the low byte is the integer's
            float far = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const float2 e = make_float2(x.element(k), x.element(k + 1));
                const float2 by = make_float2(inverse, inverse), unit = make_float2(s, s), one = make_float2(-1.0f, -1.0f), round = make_float2(kRound, kRound);
                const float2 near = fma2(e, by, round);
                if constexpr (!kBf16) {
                    const float2 rest = fma2(fma2(near, one, round), unit, e);
                    far = fmaxf(far, fmaxf(fabsf(rest.x), fabsf(rest.y)));
                }
                w[k] = __float_as_uint(near.x);
                w[k + 1] = __float_as_uint(near.y);
            }
            if (!kBf16 && 2.0f * far >= s) {
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(i8_fix(__uint_as_float(w[k]) - kRound, x.element(k), s) + kRound);
            }
            *reinterpret_cast<uint2*>(out + u * 8ll) =
                bad ? make_uint2(0, 0) : make_uint2(kv8_pack(w[0], w[1], w[2], w[3]), kv8_pack(w[4], w[5], w[6], w[7]));
        };
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
            if (u * kThreads + t < units) put(v[u], u * kThreads + t);
        for (int u = kUnits * kThreads + t; u < units; u += kThreads) {
            I8Unit<kBf16> x;
            x.load(p.x, in + u * 8ll);
            put(x, u);
        }
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
//
// 1 x 4096 x 4096 in 5.1 us (3.3 TB/s), 16 in 5.8, 8 x 14336 x 4096 in 14.9
// (4.0), 16 in 17.2, from DRAM; 16 x 4096 x 4096 and the pass that quantises its rows in 9.2 together
// (10.3 without the weights' prefetch). What is left is a chain:
// the start, two rounds of loads, the sums' meeting. All loads of a warp ahead
// of the first product took 6.6 us where two rounds took 6.2 (16 rows).
constexpr int kI8Warps = 8, kI8Ahead = 8;

template <int NT, bool kBf16>
__global__ void __launch_bounds__(32 * kI8Warps) i8_rows_kernel(I8Params p) {
    __shared__ int s_sum[kI8Warps][16][8 * NT + 1];
    // The weights are on their way to the L2 before the launch ahead has ended. This reads nothing: what that launch
    // still writes to them meets the same L2.
    if (threadIdx.x < 16 && static_cast<int>(blockIdx.x * 16 + threadIdx.x) < p.channels)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w + static_cast<size_t>(blockIdx.x * 16 + threadIdx.x) * p.w_stride), "r"(p.depth)
                     : "memory");
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
    constexpr int kAhead = kI8Ahead / NT;
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

// The last phases of a ring of `stages` barriers that was used n times, which
// nobody has waited for: no arrival is on its way when the CTA gives its
// memory back (commits arrive in any order).
__device__ __forceinline__ void mbar_settle_ring(uint32_t bars, int stages, int n) {
    for (int j = max(0, n - stages); j < n; ++j) mbar_settle(bars + 8 * (j % stages), (j / stages) & 1);
}

// Many rows: tiles on the tcgen05 tensor cores, a CTA (or a pair of them) an SM
// that takes tiles in turn. Warp 0 brings 128 bytes of depth a stage by TMA,
// warp 1 issues the products into one of two accumulators in TMEM, and warps
// 2-9 take the other one out, a row and half of the channels a thread.
//
// i8_product_kernel: 128 rows x kN channels a CTA. i8_pair_kernel: 256 x 256 a
// pair of CTAs (cta_group::2): each has 128 of the rows and 128 of the
// channels in its shared memory and the products read both, so that a CTA's
// copies are 32 KB for what takes 48 KB alone.
//
// 8192 x 16384 x 4096, bound by the tensor cores under the power limit: 363 us
// where a captured graph has a few of them (3.0 * 10^15 operations a second, 92 %
// of twice the measured bf16 rate), 418 in a long loop of calls (2.6; 95 % of
// twice the sustained rate). 1024 x 4096 x 4096 17.7 us and 512 x 4096 x 4096
// 14.3, one wave each: 0.35 to 0.45 us for 128 bytes of depth, which is what the
// copies from the L2 take (192 channels a pair, with 28 KB a stage, took 0.41
// where 256 took 0.43: dropped). Tiles of 128 x 256 by one CTA read a fifth more
// from the L2: dropped, too.
constexpr int kI8Threads = 320;
constexpr int kI8Staging = 8 * 32 * 64;  // bytes: 32 rows of 64 for each of warps 2-9

template <int kN>
__host__ __device__ constexpr int i8_stages() { return kN == 128 ? 6 : 8; }

template <int kN>
__host__ __device__ constexpr int i8_smem() { return 1024 + i8_stages<kN>() * (128 + kN) * 128 + kI8Staging; }

constexpr int kI8PairStages = 6;
constexpr int kI8PairSmem = 1024 + kI8PairStages * 256 * 128 + kI8Staging;

// Tiles in bands of kBand row tiles, so that the CTAs at work share rows and weights in the L2.
__device__ __forceinline__ void i8_place(const I8Params& p, int tile, int& m, int& n) {
    constexpr int kBand = 16;
    const int band = tile / (kBand * p.tiles_n), in = tile - band * kBand * p.tiles_n;
    const int high = min(kBand, p.tiles_m - band * kBand);
    n = in / high;
    m = band * kBand + in - n * high;
}

// Where a warp's staged row lies: 64 bytes, its 16-byte pieces turned so that
// neither a piece of every row nor a row's pieces share banks.
__device__ __forceinline__ uint32_t i8_staged(uint32_t staging, int row, int piece) {
    return staging + row * 64 + ((piece ^ (row >> 1 & 3)) * 16);
}

// The last channels of 32 staged rows that are a multiple of 16 bytes apart.
template <bool kBf16>
__device__ __forceinline__ void i8_store_last(const I8Params& p, uint32_t staging, int row0, int n0) {
    const int lane = threadIdx.x & 31, w = lane & 15, cols = p.channels - n0;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + (lane >> 4);
        const size_t to = static_cast<size_t>(row0 + r) * p.y_stride + n0;
        uint32_t mine;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(mine) : "r"(i8_staged(staging, r, w >> 2) + (w & 3) * 4));
        if (row0 + r >= p.rows) continue;
        if constexpr (kBf16) {
            uint16_t* y = static_cast<uint16_t*>(p.y) + to + 2 * w;
            if (2 * w + 1 < cols) *reinterpret_cast<uint32_t*>(y) = mine;
            else if (2 * w < cols) *y = static_cast<uint16_t>(mine);
        } else {
            if (w < cols) static_cast<uint32_t*>(p.y)[to + w] = mine;
        }
    }
}

// `cols` of the 64 bf16 or 32 fp32 columns from n0 on of 16 rows of any
// alignment, staged in 128 bytes each: a lane stores the word of y that holds
// what its word of the staged row does. bf16 rows that start between two of
// y's words are staged one element on, their first word with the last element
// of the columns before (of the first columns: not stored).
template <bool kBf16>
__device__ __forceinline__ void i8_store_words(const I8Params& p, uint32_t staging, int row0, int n0, int cols, bool first) {
    const int lane = threadIdx.x & 31, rows = p.rows - row0;
    const bool whole = lane < (kBf16 ? cols / 2 : cols), shifted = lane < (cols + 1) / 2 && !(first && lane == 0);
    const uint32_t from = staging + lane * 4;
    const long long step = p.y_stride * (kBf16 ? 2 : 4);
    const uintptr_t to = reinterpret_cast<uintptr_t>(p.y) + (static_cast<size_t>(row0) * p.y_stride + n0) * (kBf16 ? 2 : 4);
    // every other row starts alike
    uint32_t* at[2];
    bool mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uintptr_t start = to + i * step;
        at[i] = reinterpret_cast<uint32_t*>(start & ~static_cast<uintptr_t>(3)) + lane;
        mine[i] = kBf16 && start & 2 ? shifted : whole;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"((from ^ ((r & 7) * 16)) + r * 128));
        if (mine[r & 1] && r < rows) *at[r & 1] = w;
        at[r & 1] = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(at[r & 1]) + 2 * step);
    }
}

// A tile's columns [c0, c1) of a warp's 32 rows (row0 + lane; channels from n0
// on) to y through `staging`, so that a store has whole sectors whatever the
// row stride; `taken` is called once they have left TMEM. scale, bias: the
// tile's channels'; xs: the row's. failed: NaN. Rows that are a multiple of 16
// bytes apart go 64 bytes at a time; others 128, a row a store, since what they
// cost is the instructions of every store (1001 x 5003 x 2064, bf16: 21.4 us;
// two rows a store, with their alignment seen to there, 30.5; 5008 channels
// 20.0).
template <bool kBf16, typename Taken>
__device__ __forceinline__ void i8_take(const I8Params& p, uint32_t tmem, uint32_t staging, int row0, int n0, int c0, int c1,
                                        const float* scale, const float* bias, float xs, bool failed, const Taken& taken) {
    constexpr int kCols = kBf16 ? 32 : 16, kSize = kBf16 ? 2 : 4;  // 64 bytes
    const int lane = threadIdx.x & 31, row = row0 + lane;
    if (failed) xs = __int_as_float(0x7fc00000);
    float finite = 0.0f;  // NaN once a value is not
    // kCols sums, the tile's from column c on, as they lie in y
    const auto values = [&](const uint32_t* r, int c, uint32_t* out) {
#pragma unroll
        for (int k = 0; k < kCols; k += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(scale + c + k), b4 = *reinterpret_cast<const float4*>(bias + c + k);
            const float v[4] = {i8_value(static_cast<int>(r[k]), xs, s4.x, b4.x), i8_value(static_cast<int>(r[k + 1]), xs, s4.y, b4.y),
                                i8_value(static_cast<int>(r[k + 2]), xs, s4.z, b4.z), i8_value(static_cast<int>(r[k + 3]), xs, s4.w, b4.w)};
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                if constexpr (kBf16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[i], v[i + 1]);
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(&b);
                    out[(k + i) / 2] = w;
                    finite = fmaf(__uint_as_float(w << 16), 0.0f, fmaf(__uint_as_float(w & 0xffff0000u), 0.0f, finite));
                } else {
                    out[k + i] = __float_as_uint(v[i]);
                    out[k + i + 1] = __float_as_uint(v[i + 1]);
                    finite = fmaf(v[i], 0.0f, fmaf(v[i + 1], 0.0f, finite));  // (channels behind the last: sums, scale and bias 0)
                }
            }
        }
    };
    if (p.y_stride * kSize % 16 == 0) {
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
            uint32_t r[32];
            tmem_load32(tmem + c, r);
            if (c + 32 >= c1) taken();
#pragma unroll
            for (int h = 0; h < 32; h += kCols) {
                uint32_t out[16];
                values(r + h, c + h, out);
#pragma unroll
                for (int k = 0; k < 4; ++k) kv8_put16(i8_staged(staging, lane, k), out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
                __syncwarp();
                const int cols = p.channels - (n0 + c + h);
                if (cols >= kCols) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int to = 8 * i + (lane >> 2);
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                                     : "r"(i8_staged(staging, to, lane & 3)));
                        if (row0 + to < p.rows)
                            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.y) + (static_cast<size_t>(row0 + to) * p.y_stride + n0 + c + h) * kSize + (lane & 3) * 16) = w;
                    }
                } else if (cols > 0) {
                    i8_store_last<kBf16>(p, staging, row0, n0 + c + h);
                }
                __syncwarp();
            }
        }
    } else {
        constexpr int kUnit = 2 * kCols;
        uint16_t* y = static_cast<uint16_t*>(p.y) + static_cast<size_t>(row) * p.y_stride + n0;
        const bool odd = kBf16 && (row * p.y_stride + n0) & 1;
        uint32_t before = 0;  // the last two elements
#pragma unroll 1
        for (int c = c0; c < c1; c += kUnit) {
            uint32_t out[32];
#pragma unroll
            for (int h = 0; h < kUnit; h += 32) {
                if (c + h < c1) {
                    uint32_t r[32];
                    tmem_load32(tmem + c + h, r);
#pragma unroll
                    for (int k = 0; k < 32; k += kCols) values(r + k, c + h + k, out + (h + k) * kSize / 4);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) out[16 + k] = 0;
                }
            }
            if (c + kUnit >= c1) taken();
            const int cols = min(min(kUnit, c1 - c), p.channels - (n0 + c));
            if (cols <= 0) continue;
            const bool ends = c + kUnit >= c1 || n0 + c + kUnit >= p.channels;
            if constexpr (kBf16) {
                if (odd && c == c0 && row < p.rows) y[c] = static_cast<uint16_t>(out[0]);
                const uint32_t last = out[31], pick = odd ? 0x5432 : 0x7654;
#pragma unroll
                for (int k = 31; k > 0; --k) out[k] = __byte_perm(out[k - 1], out[k], pick);
                out[0] = __byte_perm(before, out[0], pick);
                before = last;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t own = staging + (lane & 15) * 128;
                if (lane >> 4 == half)
#pragma unroll
                    for (int k = 0; k < 8; ++k) kv8_put16(own + ((k ^ (lane & 7)) * 16), out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
                __syncwarp();
                i8_store_words<kBf16>(p, staging, row0 + 16 * half, n0 + c, cols, c == c0);
                if (kBf16 && ends && lane >> 4 == half && (cols + odd) % 2 && row < p.rows) {  // half a word is left
                    const int w = (cols + odd) / 2;
                    uint32_t left = before >> 16;
                    if (w < 32) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(left) : "r"(own + (((w >> 2) ^ (lane & 7)) * 16) + (w & 3) * 4));
                    y[c + cols - 1] = static_cast<uint16_t>(left);
                }
                __syncwarp();
            }
        }
    }
    if (row < p.rows && finite != 0.0f) {
        if (failed) {
            if (p.status) atomicMax(p.status + row, kStatusDevice);
        } else {
            flag_nonfinite(p.status, row);
        }
    }
}

// What the threads of warps 2-9 read of scales and biases for a tile: each a
// channel's and its row's, one tile ahead.
template <int kN>
struct I8Scales {
    float channel, bias, row;
    __device__ __forceinline__ void load(const I8Params& p, int own_row, int n0) {
        const int n = n0 + static_cast<int>(threadIdx.x) - 64;
        const bool in = static_cast<int>(threadIdx.x) - 64 < kN && n < p.channels;
        channel = in ? p.w_scales[n] : 0.0f;
        bias = in && p.bias ? p.bias[n] : 0.0f;
        row = own_row < p.rows ? p.x_scales[own_row] : 0.0f;
    }
    // the channels' to all of those warps
    __device__ __forceinline__ void share(float* scales, float* biases) const {
        const int c = static_cast<int>(threadIdx.x) - 64;
        if (c < kN) {
            scales[c] = channel;
            biases[c] = bias;
        }
        __syncwarp();
        asm volatile("bar.sync 1, 256;" ::: "memory");
    }
};

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
            mbar_init(drained + 8 * a, 8);
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
    pdl_wait();
    pdl_trigger();
    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
            int m, n;
            i8_place(p, tile, m, n);
            for (int k = 0; k < nk; ++k, ++it) {
                const int s = it % kStages;
                if (it >= kStages && !(ok = mbar_wait(empty + 8 * s, (it / kStages - 1) & 1, nullptr, &s_failed))) break;
                mbar_expect_tx(full + 8 * s, kStageBytes);
                tma_load_2d(stages + s * kStageBytes, &tm_x, k * 128, m * 128, full + 8 * s);
                tma_load_2d(stages + s * kStageBytes + 128 * 128, &tm_w, k * 128, n * kN, full + 8 * s);
            }
        }
        if (!ok)  // a wait ran out: no copy is on its way when the CTA gives its memory back
            mbar_settle_ring(full, kStages, it);
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
        if (ok) mbar_settle_ring(empty, kStages, it);
    } else if (warp >= 2) {
        const int quarter = warp & 3;
        int turn = 0, m = 0, n = 0;
        I8Scales<kN> scales{};
        const auto ahead = [&](int tile) {
            i8_place(p, tile, m, n);
            scales.load(p, m * 128 + quarter * 32 + lane, n * kN);
        };
        if (static_cast<int>(blockIdx.x) < tiles) ahead(blockIdx.x);
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
            const int a = turn & 1, row0 = m * 128 + quarter * 32, n0 = n * kN;
            const float xs = scales.row;
            scales.share(s_scale[a], s_bias[a]);
            if (tile + static_cast<int>(gridDim.x) < tiles) ahead(tile + gridDim.x);
            mbar_wait(done + 8 * a, (turn / 2) & 1, nullptr, &s_failed);
            __syncwarp();
            const bool failed = __any_sync(kFull, *static_cast<volatile int*>(&s_failed));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int c0 = (warp - 2) / 4 * (kN / 2);
            i8_take<kBf16>(p, tmem + a * kN + (static_cast<uint32_t>(quarter * 32) << 16), stages + kStages * kStageBytes + (warp - 2) * 2048,
                           row0, n0, c0, c0 + kN / 2, s_scale[a], s_bias[a], xs, failed, [&] {
                               asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                               __syncwarp();
                               if (lane == 0) mbar_arrive(drained + 8 * a);
                           });
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

__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {  // the same place in a CTA of the cluster
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Few tiles: the depth of one is split over the CTAs of a cluster, whose sums
// meet in shared memory (integers: the result does not depend on the split).
// Bound by the weights' way to few CTAs and then by the meeting (3.3 us with 64
// channels a tile, 4.5 with 128): 512 x 512 x 2048 in 7.1 us (a CTA a tile:
// 8.2), 32 and 128 x 4096 x 4096 in 9.2 and 11.6 (13.4, 13.7).
template <int kN>
__host__ __device__ constexpr int i8_split_stages() { return kN == 128 ? 6 : 8; }

template <int kN, bool kBf16>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_split_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, I8Params p) {
    constexpr int kStages = i8_split_stages<kN>(), kStageBytes = (128 + kN) * 128, kPitch = kN * 4 + 16;
    static_assert(128 * kPitch <= kStages * kStageBytes, "the sums outgrow the operands' room");
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * kStages + 1];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    const uint32_t stages = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = smem_addr(s_bars), empty = full + 8 * kStages, done = empty + 8 * kStages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank, splits;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(done, 1);
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(kN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    int m, n;
    i8_place(p, static_cast<int>(blockIdx.x / splits), m, n);
    const int nk = (p.depth + 127) / 128, per = (nk + static_cast<int>(splits) - 1) / static_cast<int>(splits);
    const int first = static_cast<int>(rank) * per, turns = min(nk, first + per) - first;  // (at least one: by the choice of this kernel)
    pdl_wait();
    pdl_trigger();
    if (warp == 0 && lane == 0) {
        int k = 0;
        bool ok = true;
        for (; k < turns; ++k) {
            const int s = k % kStages;
            if (k >= kStages && !(ok = mbar_wait(empty + 8 * s, (k / kStages - 1) & 1, nullptr, &s_failed))) break;
            mbar_expect_tx(full + 8 * s, kStageBytes);
            tma_load_2d(stages + s * kStageBytes, &tm_x, (first + k) * 128, m * 128, full + 8 * s);
            tma_load_2d(stages + s * kStageBytes + 128 * 128, &tm_w, (first + k) * 128, n * kN, full + 8 * s);
        }
        if (!ok)  // a wait ran out: no copy is on its way when the CTA gives its memory back
            mbar_settle_ring(full, kStages, k);
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = umma_idesc_i8(128, kN);
        bool ok = true;
        for (int k = 0; k < turns; ++k) {
            const int s = k % kStages;
            if (!(ok = mbar_wait(full + 8 * s, (k / kStages) & 1, nullptr, &s_failed))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = stages + s * kStageBytes;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                umma_i8(tmem, umma_desc_sw128(at + kk * 32), umma_desc_sw128(at + 128 * 128 + kk * 32), idesc, (k | kk) != 0);
            umma_commit(empty + 8 * s);
        }
        umma_commit(done);
        mbar_settle(done, 0);  // nor is a product
        if (ok) mbar_settle_ring(empty, kStages, turns);
    }
    __syncwarp();
    mbar_wait(done, 0, nullptr, &s_failed);
    __syncthreads();  // every copy has been multiplied: the operands' room takes the sums
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp >= 2 && warp < 6) {
        const int quarter = warp & 3;
        const uint32_t to = stages + (quarter * 32 + lane) * kPitch;
#pragma unroll
        for (int c = 0; c < kN; c += 32) {
            uint32_t r[32];
            tmem_load32(tmem + c + (static_cast<uint32_t>(quarter * 32) << 16), r);
#pragma unroll
            for (int k = 0; k < 32; k += 4) kv8_put16(to + (c + k) * 4, r[k], r[k + 1], r[k + 2], r[k + 3]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_meet();
    // rows rank, rank + splits, ... of the tile; four channels a thread
    constexpr int kQuads = kN / 4;
    const int rows = min(128, p.rows - m * 128);
    for (int x = threadIdx.x; x < 128 / static_cast<int>(splits) * kQuads; x += kI8Threads) {
        const int r = x / kQuads * static_cast<int>(splits) + static_cast<int>(rank), c = x % kQuads * 4;
        if (r >= rows) continue;
        int4 sum = make_int4(0, 0, 0, 0);
        int bad = 0;
        for (uint32_t peer = 0; peer < splits; ++peer) {
            int4 v;
            int f;
            asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(cluster_addr(stages + r * kPitch + c * 4, peer)) : "memory");
            asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(f) : "r"(cluster_addr(smem_addr(&s_failed), peer)) : "memory");
            sum = make_int4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
            bad |= f;
        }
        const int row = m * 128 + r, n0 = n * kN + c;
        const float xs = bad ? __int_as_float(0x7fc00000) : p.x_scales[row];
        const int v[4] = {sum.x, sum.y, sum.z, sum.w};
        const size_t at = static_cast<size_t>(row) * p.y_stride + n0;
        float y[4];
        bool finite = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = n0 + k < p.channels;
            y[k] = in ? i8_value(v[k], xs, p.w_scales[n0 + k], p.bias ? p.bias[n0 + k] : 0.0f) : 0.0f;
            finite &= isfinite(kBf16 ? __bfloat162float(__float2bfloat16(y[k])) : y[k]);
        }
        if (p.y_stride % 4 == 0 && n0 + 4 <= p.channels) {
            store_row4<kBf16>(p.y, at, make_float4(y[0], y[1], y[2], y[3]));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n0 + k < p.channels) i8_store<kBf16>(p.y, at + k, y[k]);
        }
        if (bad && p.status) atomicMax(p.status + row, kStatusDevice);
        else if (!finite) flag_nonfinite(p.status, row);
    }
    __syncwarp();  // (rows behind the last and lanes with other stores end their turns apart)
    cluster_meet();  // no CTA's sums go while another reads them
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kN) : "memory");
    }
}

// mbar_wait for a barrier that the cluster's other CTA arrives at, too.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* cta_failed) {
    const long long start = clock64();
    while (true) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (*cta_failed) return false;
        if (clock64() - start > kWaitBudgetCycles) {
            *cta_failed = 1;
            return false;
        }
    }
}

template <bool kBf16>
__global__ void __launch_bounds__(kI8Threads, 1) __cluster_dims__(2, 1, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, I8Params p) {
    constexpr int kN = 256, kStages = kI8PairStages, kStageBytes = 256 * 128;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[2 * kStages + 5];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(16) float s_scale[2][kN], s_bias[2][kN];
    const uint32_t stages = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = smem_addr(s_bars), empty = full + 8 * kStages, done = empty + 8 * kStages, drained = done + 16, idle = drained + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;  // 0 leads: its barriers count both CTAs' copies, its thread issues the products
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(done + 8 * a, 1);
            mbar_init(drained + 8 * a, 16);
        }
        mbar_init(idle, 1);
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(2 * kN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_meet();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    const int nk = (p.depth + 127) / 128, tiles = p.tiles_m * p.tiles_n, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    pdl_wait();
    pdl_trigger();
    if (warp == 0 && lane == 0) {
        const uint32_t lead_full = cluster_addr(full, 0);
        int it = 0;
        bool ok = true;
        for (int tile = first; ok && tile < tiles; tile += step) {
            int m, n;
            i8_place(p, tile, m, n);
            for (int k = 0; k < nk; ++k, ++it) {
                const int s = it % kStages;
                if (it >= kStages && !(ok = mbar_wait_cluster(empty + 8 * s, (it / kStages - 1) & 1, &s_failed))) break;
                if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * kStageBytes);
                const auto copy = [&](uint32_t to, const CUtensorMap* map, int row) {
                    asm volatile(
                        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
                        ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(lead_full + 8 * s), "r"(k * 128), "r"(row)
                        : "memory");
                };
                copy(stages + s * kStageBytes, &tm_x, m * 256 + rank * 128);
                copy(stages + s * kStageBytes + 128 * 128, &tm_w, n * kN + rank * 128);
            }
        }
        // A wait ran out: copies that are on their way end in much less than this.
        if (!ok)
            for (const long long since = clock64(); clock64() - since < kWaitBudgetCycles / 1024;) __nanosleep(1000);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t idesc = umma_idesc_i8(256, kN);
        const auto commit = [&](uint32_t bar) {  // in both CTAs
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                         "h"(static_cast<uint16_t>(3))
                         : "memory");
        };
        int it = 0, turn = 0;
        bool ok = true;
        for (int tile = first; ok && tile < tiles; tile += step, ++turn) {
            const int a = turn & 1;
            if (turn >= 2 && !(ok = mbar_wait_cluster(drained + 8 * a, (turn / 2 - 1) & 1, &s_failed))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int k = 0; k < nk; ++k, ++it) {
                const int s = it % kStages;
                if (!(ok = mbar_wait_cluster(full + 8 * s, (it / kStages) & 1, &s_failed))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = stages + s * kStageBytes;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    asm volatile(
                        "{\n\t.reg .pred p;\n\t"
                        "setp.ne.b32 p, %4, 0;\n\t"
                        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                        ::"r"(tmem + a * kN), "l"(umma_desc_sw128(at + kk * 32)), "l"(umma_desc_sw128(at + 128 * 128 + kk * 32)), "r"(idesc),
                        "r"(static_cast<uint32_t>((k | kk) != 0))
                        : "memory");
                commit(empty + 8 * s);
            }
            if (ok) commit(done + 8 * a);
        }
        commit(idle);  // no product is on its way when the CTAs give their memory back
        mbar_settle(idle, 0);
        if (ok) mbar_settle_ring(empty, kStages, it);
    } else if (warp >= 2) {
        const int quarter = warp & 3;
        const uint32_t lead_drained = cluster_addr(drained, 0);
        int turn = 0, m = 0, n = 0;
        I8Scales<kN> scales{};
        const auto ahead = [&](int tile) {
            i8_place(p, tile, m, n);
            scales.load(p, m * 256 + static_cast<int>(rank) * 128 + quarter * 32 + lane, n * kN);
        };
        if (first < tiles) ahead(first);
        for (int tile = first; tile < tiles; tile += step, ++turn) {
            const int a = turn & 1, row0 = m * 256 + static_cast<int>(rank) * 128 + quarter * 32, n0 = n * kN;
            const float xs = scales.row;
            scales.share(s_scale[a], s_bias[a]);
            if (tile + step < tiles) ahead(tile + step);
            mbar_wait_cluster(done + 8 * a, (turn / 2) & 1, &s_failed);
            __syncwarp();
            const bool failed = __any_sync(kFull, *static_cast<volatile int*>(&s_failed));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int c0 = (warp - 2) / 4 * (kN / 2);
            i8_take<kBf16>(p, tmem + a * kN + (static_cast<uint32_t>(quarter * 32) << 16), stages + kStages * kStageBytes + (warp - 2) * 2048,
                           row0, n0, c0, c0 + kN / 2, s_scale[a], s_bias[a], xs, failed, [&] {
                               asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                               __syncwarp();
                               if (lane == 0)
                                   asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_drained + 8 * a) : "memory");
                           });
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // What the other CTA has committed here: not before the last tile has been taken out, however long that took.
    if (rank != 0 && warp == 1) {  // a barrier a lane
        const int j = (tiles - first + step - 1) / step * nk - lane;  // of the ring, from its last turn back
        if (lane == 0) mbar_settle(idle, 0);
        else if (lane <= kStages && j >= 0 && !*static_cast<volatile int*>(&s_failed)) mbar_settle(empty + 8 * (j % kStages), (j / kStages) & 1);
    }
    __syncwarp();
    cluster_meet();  // neither CTA's memory goes while the other may reach it
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * kN) : "memory");
    }
}

}  // namespace phonon
