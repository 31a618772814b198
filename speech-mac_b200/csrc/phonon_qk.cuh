// RMS norm of every query and key head with the position rotation in the same
// pass (sm_100a).
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head; skipped without w)
//   (a, b) -> (a cos - b sin, a sin + b cos)   angle = position * theta^(-2i / rotary_dim)
//
// for the rotary_dim / 2 pairs of a head: (2i, 2i + 1), or (i, i + rotary_dim
// / 2). Bound by the bytes of the rows, read once and written once. A warp
// takes one row's heads (or a slice of them) in turn: a lane owns 4 dims of a
// head, so its angles, weights and frequencies stay in registers for all
// heads of the row, and the two halves of a pair meet by a shuffle.
//
// The angle is reduced in turns: position * theta^(...) / 2 pi and its nearest
// integer in 64 bits, the remainder (within half a turn) rounded to 32, an
// error below 2^-25 turns at any position; sine and cosine are sincospif's.
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

template <int D, bool kBf16, bool kHalves>
__global__ void __launch_bounds__(128) qk_norm_rope_kernel(QkParams p) {
    constexpr int kLanes = D / 4, kPerWarp = 32 / kLanes;  // lanes of a head, heads of a warp pass
    constexpr int kAngles = kHalves ? 4 : 2;
    const int lane = threadIdx.x & 31, sub = lane / kLanes, d = (lane % kLanes) * 4;
    const int half = p.rotary / 2;
    // the lane's frequencies, in turns per position
    double turns[kAngles];
#pragma unroll
    for (int k = 0; k < kAngles; ++k) {
        const int i = kHalves ? (d < half ? d + k : d + k - half) : d / 2 + k;
        turns[k] = exp2(-2.0 * i / p.rotary * p.log2_theta) * 0.15915494309189533577;
    }
    pdl_wait();
    pdl_trigger();
    float4 w[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
        w[s] = p.weight[s] ? __ldg(reinterpret_cast<const float4*>(p.weight[s] + d)) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    const int total = p.heads[0] + p.heads[1];
    const int passes = (total + kPerWarp - 1) / kPerWarp, per = (passes + p.slices - 1) / p.slices;
    const long long items = static_cast<long long>(p.rows) * p.slices;
    const long long stride = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
    for (long long item = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items;
         item += stride) {
        const int row = static_cast<int>(item / p.slices), slice = static_cast<int>(item % p.slices);
        const int position = __ldg(p.positions + row);
        float sn[kAngles], cs[kAngles];
#pragma unroll
        for (int k = 0; k < kAngles; ++k) {
            const double t = position * turns[k];
            sincospif(2.0f * static_cast<float>(t - rint(t)), &sn[k], &cs[k]);
        }
        bool finite = true;
        for (int u = slice * per; u < min(passes, (slice + 1) * per); ++u) {
            const int h = u * kPerWarp + sub;
            const bool live = h < total;
            const int side = live && h >= p.heads[0] ? 1 : 0;
            const size_t at = static_cast<size_t>(side ? h - p.heads[0] : h) * D + d;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live) x = load_row4<kBf16>(p.in[side], row * static_cast<size_t>(p.in_stride[side]) + at);
            // every lane takes part in the shuffles: a pass can hold normed and plain heads
            float sq = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, x.w * x.w)));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(kFull, sq, o);
            if (p.weight[side]) {
                const float r = __fdiv_rn(1.0f, __fsqrt_rn(fmaf(sq, 1.0f / D, p.epsilon)));
                const float4 v = side ? w[1] : w[0];
                x = make_float4(x.x * r * v.x, x.y * r * v.y, x.z * r * v.z, x.w * r * v.w);
            }
            if constexpr (kHalves) {
                const int from = d < half ? lane + half / 4 : lane - half / 4;
                const float4 o = make_float4(__shfl_sync(kFull, x.x, from), __shfl_sync(kFull, x.y, from),
                                             __shfl_sync(kFull, x.z, from), __shfl_sync(kFull, x.w, from));
                if (d < half)
                    x = make_float4(x.x * cs[0] - o.x * sn[0], x.y * cs[1] - o.y * sn[1], x.z * cs[2] - o.z * sn[2],
                                    x.w * cs[3] - o.w * sn[3]);
                else if (d < p.rotary)
                    x = make_float4(o.x * sn[0] + x.x * cs[0], o.y * sn[1] + x.y * cs[1], o.z * sn[2] + x.z * cs[2],
                                    o.w * sn[3] + x.w * cs[3]);
            } else {
                if (d < p.rotary) {
                    const float a = x.x, b = x.y;
                    x.x = a * cs[0] - b * sn[0];
                    x.y = a * sn[0] + b * cs[0];
                }
                if (d + 2 < p.rotary) {
                    const float a = x.z, b = x.w;
                    x.z = a * cs[1] - b * sn[1];
                    x.w = a * sn[1] + b * cs[1];
                }
            }
            if (live) {
                finite &= isfinite(x.x) & isfinite(x.y) & isfinite(x.z) & isfinite(x.w);
                store_row4<kBf16>(p.out[side], row * static_cast<size_t>(p.out_stride[side]) + at, x);
            }
        }
        if (p.status && !__all_sync(kFull, finite) && lane == 0) flag_nonfinite(p.status, row);
    }
}

}  // namespace phonon
