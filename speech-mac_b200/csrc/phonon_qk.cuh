// RMS norm of every query and key head with the position rotation in the same
// pass (sm_100a).
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head; skipped without w)
//   (a, b) -> (a cos - b sin, a sin + b cos)   angle = position * theta^(-2i / rotary_dim)
//
// for the rotary_dim / 2 pairs of a head: (2i, 2i + 1), or (i, i + rotary_dim
// / 2). Bound by the bytes of the rows, read once and written once. A warp
// takes rows (or slices of a row's heads, where rows are few) in turn; a lane
// owns 8 dims of a head in two chunks of 4, both values of every pair among
// them, so that the rotation needs no exchange and the row's four sines and
// the weights stay in registers for all its heads. The next kAhead passes, of the next row if need be, are
// on their way while kAhead are worked on side by side.
//
// The angle in turns is position * theta^(...) / 2 pi modulo 1. The frequency
// is held as a 64-bit fraction of a turn (from double, within 2^-55), so that
// the product with the position wraps at whole turns by itself: an error below
// 2^-33 turns up to position 2^22, 2^-24 at the last position of 31 bits; its
// upper 32 bits, signed, go to fp32 (2^-25 turns) and sincospif.
//
// Measured on B200 (34 us a pass, 4.9 TB/s, 76 % of the copy rate, for 8192
// rows of 32 + 8 heads of 128 in bf16; 57.6 us, 5.8 TB/s in fp32): bf16 rows are
// bound by instructions (about 100 a pass of two heads), fp32 rows by the
// DRAM. Dims of a pair in different lanes (a shuffle each, twice the sines)
// took 43 us, one CTA a row with its sines in shared memory 94 us (their 64-bit
// powers once a row), no loads ahead 64 us.
#pragma once

#include "phonon_kv8.cuh"

namespace phonon {

struct QkParams {
    const void* in[2];  // queries, keys: rows `stride` elements apart
    void* out[2];
    long long in_stride[2], out_stride[2];
    const float* weight[2];  // [D] or null
    const int32_t* positions;
    int32_t* status;  // [rows] or null
    int rows, heads[2], rotary, slices;
    float epsilon;
    double log2_theta;
};

template <int D, bool kBf16, bool kHalves, int kAhead, int kCtas>
__global__ void __launch_bounds__(128, kCtas) qk_norm_rope_kernel(QkParams p) {
    constexpr int kLanes = D / 8, kPerWarp = 32 / kLanes;  // lanes of a head, heads of a warp pass
    constexpr int kSize = kBf16 ? 2 : 4;
    using Raw = std::conditional_t<kBf16, uint2, uint4>;
    const int lane = threadIdx.x & 31, sub = lane / kLanes, l = lane % kLanes;
    // dims [chunk[0], + 4) and [chunk[1], + 4): halves are paired across the chunks, neighbours within
    const int half = p.rotary / 2;
    const bool turned = kHalves && l < p.rotary / 8;
    const int chunk[2] = {turned ? 4 * l : 8 * l, turned ? half + 4 * l : 8 * l + 4};
    unsigned long long turns[4];  // per position, 2^-64 of a turn
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int i = kHalves ? chunk[0] + k : chunk[0] / 2 + k;
        const double t = exp2(-2.0 * i / p.rotary * p.log2_theta) * 0.15915494309189533577;
        turns[k] = __double2ull_rn((t - floor(t)) * 18446744073709551616.0);
    }
    pdl_wait();
    pdl_trigger();
    float w[2][8];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float4 v = p.weight[s] ? *reinterpret_cast<const float4*>(p.weight[s] + chunk[c]) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
            w[s][4 * c] = v.x, w[s][4 * c + 1] = v.y, w[s][4 * c + 2] = v.z, w[s][4 * c + 3] = v.w;
        }
    // passes of the queries, then of the keys: a pass has one side
    const int pass_q = (p.heads[0] + kPerWarp - 1) / kPerWarp, passes = pass_q + (p.heads[1] + kPerWarp - 1) / kPerWarp;
    const int per = (passes + p.slices - 1) / p.slices;
    const int items = p.rows * p.slices, stride = gridDim.x * (blockDim.x >> 5);
    int item = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (item >= items) return;  // the whole warp
    const float smallest = p.epsilon < 1e-25f ? 1e-25f : 0.0f;  // sums below lose bits that count
    Raw raw[kAhead][2];
    // the passes [u, min(u + kAhead, the side's end, stop)) of a row
    auto load = [&](int row, int u, int stop) {
        const bool side = u >= pass_q;
        const int h0 = (u - (side ? pass_q : 0)) * kPerWarp + sub, heads = side ? p.heads[1] : p.heads[0];
        const char* in = static_cast<const char*>(side ? p.in[1] : p.in[0]) +
                         row * (side ? p.in_stride[1] : p.in_stride[0]) * kSize + h0 * (D * kSize);
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                raw[a][c] = Raw{};
                if (u + a < stop && h0 + a * kPerWarp < heads)
                    raw[a][c] = *reinterpret_cast<const Raw*>(in + a * (kPerWarp * D * kSize) + chunk[c] * kSize);
            }
    };
    auto end_of = [&](int u, int stop) { return min(min(u + kAhead, stop), u < pass_q ? pass_q : passes); };
    int row = item / p.slices, first = (item - row * p.slices) * per;
    int position = p.positions[row];
    if (first < passes) load(row, first, min(passes, first + per));
    while (true) {
        const int stop = min(passes, first + per);
        const int next = item + stride, next_row = next < items ? next / p.slices : row;
        const int next_first = (next - next_row * p.slices) * per;
        const int next_position = p.positions[next_row];
        float sn[8], cs[8];  // of every dim, with the sign of its own term: a cos - b sin, a sin + b cos
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned long long t = static_cast<unsigned long long>(static_cast<long long>(position)) * turns[k];
            float s, c;
            sincospif(static_cast<float>(static_cast<int>(t >> 32)) * 0x1p-31f, &s, &c);
            if (kHalves ? !turned : chunk[0] + 2 * k >= p.rotary) s = 0.0f, c = 1.0f;
            const int one = kHalves ? k : 2 * k, two = kHalves ? k + 4 : 2 * k + 1;
            sn[one] = -s;
            sn[two] = s;
            cs[one] = cs[two] = c;
        }
        float finite = 0.0f;  // NaN once an output, rounded, is not
        __nv_bfloat162 finite2 = __floats2bfloat162_rn(0.0f, 0.0f);
        int u = first;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int side_end = min(stop, side ? passes : pass_q), heads = p.heads[side];
            if (u >= side_end) continue;
            constexpr int kOther = kHalves ? 4 : 1;  // a dim's pair: k ^ kOther
            float a0[8], a1[8];                      // y = r (a0 x + a1 other)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                a0[k] = cs[k] * w[side][k];
                a1[k] = sn[k] * w[side][k ^ kOther];
            }
            char* out = static_cast<char*>(p.out[side]) + row * p.out_stride[side] * kSize;
            for (; u < side_end; u += kAhead) {
                float x[kAhead][8], sq[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    sq[a] = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t* words = reinterpret_cast<const uint32_t*>(&raw[a][k / 4]);
                        x[a][k] = __uint_as_float(!kBf16 ? words[k % 4] : k % 2 ? words[k % 4 / 2] & 0xffff0000u : words[k % 4 / 2] << 16);
                        sq[a] = fmaf(x[a][k], x[a][k], sq[a]);
                    }
                }
                const int after = end_of(u, stop);
                if (after < stop) load(row, after, stop);
                else if (next < items && next_first < passes) load(next_row, next_first, min(passes, next_first + per));
                // every lane takes part in the shuffles
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) sq[a] += __shfl_xor_sync(kFull, sq[a], o);
                const int h0 = (u - (side ? pass_q : 0)) * kPerWarp + sub;
                float inverse[kAhead], most = 0.0f, least = 1.0f;
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    inverse[a] = rsqrtf(fmaf(sq[a], 1.0f / D, p.epsilon));
                    most = fmaxf(most, sq[a]);
                    least = fminf(least, sq[a]);
                }
                // squares outside fp32's range: of x times a power of two
                if (__any_sync(kFull, !(most < 1e37f) || least < smallest)) {
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) {
                        const float by = sq[a] < 1.0f ? 0x1p+64f : 0x1p-64f;
                        float again = 0.0f;
#pragma unroll
                        for (int k = 0; k < 8; ++k) again = fmaf(x[a][k] * by, x[a][k] * by, again);
#pragma unroll
                        for (int o = kLanes / 2; o > 0; o >>= 1) again += __shfl_xor_sync(kFull, again, o);
                        if (!(sq[a] < 1e37f) || sq[a] < smallest) inverse[a] = rsqrtf(fmaf(again, 1.0f / D, p.epsilon * by * by)) * by;
                    }
                }
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    // (0 where the pass has no head: its x is 0, and without an epsilon so is the mean)
                    const bool there = u + a < side_end && h0 + a * kPerWarp < heads;
                    const float r = !there ? 0.0f : p.weight[side] ? inverse[a] : 1.0f;
                    float y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[a][k] *= r;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        y[k] = fmaf(x[a][k], a0[k], x[a][k ^ kOther] * a1[k]);
                        if constexpr (!kBf16) finite = fmaf(y[k], 0.0f, finite);
                    }
                    Raw packed[2];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t* words = reinterpret_cast<uint32_t*>(&packed[k / 4]);
                        if constexpr (!kBf16) {
                            words[k % 4] = __float_as_uint(y[k]);
                        } else if (k % 2 == 0) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(y[k], y[k + 1]);
                            words[k % 4 / 2] = *reinterpret_cast<const uint32_t*>(&b);
                            finite2 = __hfma2(b, __floats2bfloat162_rn(0.0f, 0.0f), finite2);
                        }
                    }
                    if (there) {
                        char* to = out + (h0 + a * kPerWarp) * (D * kSize);
                        *reinterpret_cast<Raw*>(to + chunk[0] * kSize) = packed[0];
                        *reinterpret_cast<Raw*>(to + chunk[1] * kSize) = packed[1];
                    }
                }
            }
            u = side_end;
        }
        if constexpr (kBf16) finite = __low2float(finite2) + __high2float(finite2);
        if (p.status && !__all_sync(kFull, finite == 0.0f) && lane == 0) flag_nonfinite(p.status, row);
        if (next >= items) break;
        item = next;
        row = next_row;
        first = next_first;
        position = next_position;
    }
}

}  // namespace phonon
