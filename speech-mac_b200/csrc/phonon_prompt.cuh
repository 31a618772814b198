// Causal attention over packed prompts (sm_100a): the row at position p of a
// prompt sees its positions (p - window, p], all up to p without a window.
//
//   out[p] = sum_j softmax_j(scale q[p] . k[j]) v[j]
//
// Rows lie packed, prompt i in rows [row_begin[i], row_begin[i + 1]), and
// query heads are grouped on K/V heads.
#pragma once

#include "phonon_kv8_prompt.cuh"

namespace phonon {

struct PromptParams {
    const void *q, *k, *v;  // [rows][heads][D], [rows][kv_heads][D] twice; rows `stride` elements apart
    void* out;
    long long q_stride, k_stride, v_stride, out_stride;
    const int32_t* begin;  // [prompts + 1]
    int32_t* status;       // [prompts] or null
    int prompts, rows, max_rows, heads, kv_heads;
    Kv8Div group;  // query heads of a K/V head
    int window;    // 0: none
    float scale;   // times log2(e)
    int tokens;    // positions of a tile
    Kv8Div by_heads;  // CTAs of a tile
};

__device__ __forceinline__ void prompt_flag(const PromptParams& p, int i, int code) {
    if (p.status) atomicMax(p.status + i, code);
}

// The slot-th tile of the call: `tokens` positions of a prompt, the last ones
// first (they see most). index < 0: the call has fewer tiles.
struct PromptTile {
    int index, row0, length, first;  // prompt, its first row and rows, the tile's first position
};

// A prompt whose rows lie outside the call's, are more than max_rows or begin
// before an earlier prompt's has none: tiles never share rows, and there are at
// most rows / tokens + prompts of them, one less for every prompt without.
// `report`: one CTA of the last slot, which reads all prompts if there is such
// a one.
template <int kThreads>
__device__ __forceinline__ PromptTile prompt_tile(const PromptParams& p, int slot, bool report) {
    constexpr int kWarps = kThreads / 32;
    __shared__ int s_count[kWarps], s_most[kWarps], s_tile[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) s_tile[0] = -1;
    int before = 0, most = 0;  // tiles and the largest begin of the prompts so far
    for (int base = 0; base < p.prompts; base += kThreads) {
        const int i = base + static_cast<int>(threadIdx.x);
        const bool there = i < p.prompts;
        const int b = there ? p.begin[i] : 0, e = there ? p.begin[i + 1] : 0;
        int top = b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(kFull, top, o);
            if (lane >= o) top = max(top, x);
        }
        if (lane == 31) s_most[warp] = top;
        __syncthreads();
        int earlier = most;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) earlier = max(earlier, s_most[w]);
            most = max(most, s_most[w]);
        }
        const bool good = b >= max(top, earlier) && e >= b && e <= p.rows && e - b <= p.max_rows;
        if (there && !good && report) prompt_flag(p, i, kStatusInvalid);
        const int tiles = there && good ? (e - b + p.tokens - 1) / p.tokens : 0;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(kFull, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) s_count[warp] = sum;
        __syncthreads();
        int ahead = before;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) ahead += s_count[w];
            before += s_count[w];
        }
        const int at = slot - (ahead + sum - tiles);
        if (at >= 0 && at < tiles) {
            s_tile[0] = i;
            s_tile[1] = b;
            s_tile[2] = e - b;
            s_tile[3] = (tiles - 1 - at) * p.tokens;
        }
        if (slot < before) break;  // the same for every thread
    }
    __syncthreads();
    return {s_tile[0], s_tile[1], s_tile[2], s_tile[3]};
}

// One row by a warp in fp32, position after position: D / 32 dims a lane.
template <int D, bool kBf16>
__device__ __forceinline__ void prompt_row(const PromptParams& p, const PromptTile& t, int position, int head, bool& finite) {
    constexpr int kDims = D / 32;
    const int lane = threadIdx.x & 31, kv_head = static_cast<int>(kv8_div(head, p.group));
    auto load = [&](const void* base, size_t at, float (&x)[kDims]) {
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            if constexpr (kBf16) x[d] = __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(base)[at + d * 32 + lane]) << 16);
            else x[d] = static_cast<const float*>(base)[at + d * 32 + lane];
        }
    };
    float q[kDims], o[kDims], m = -INFINITY, l = 0.0f;
    load(p.q, static_cast<size_t>(t.row0 + position) * p.q_stride + static_cast<size_t>(head) * D, q);
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] = 0.0f;
    for (int j = p.window ? max(0, position - p.window + 1) : 0; j <= position; ++j) {
        float k[kDims], v[kDims], s = 0.0f;
        load(p.k, static_cast<size_t>(t.row0 + j) * p.k_stride + static_cast<size_t>(kv_head) * D, k);
        load(p.v, static_cast<size_t>(t.row0 + j) * p.v_stride + static_cast<size_t>(kv_head) * D, v);
#pragma unroll
        for (int d = 0; d < kDims; ++d) s = fmaf(q[d], k[d], s);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(kFull, s, w);
        s *= p.scale;
        const float now = isnan(s) ? s : fmaxf(m, s);
        const float by = m == now ? 1.0f : ex2(m - now), w = s == -INFINITY && now == -INFINITY ? 0.0f : ex2(s - now);
        m = now;
        l = fmaf(l, by, w);
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] = fmaf(o[d], by, w * v[d]);
    }
    const size_t at = static_cast<size_t>(t.row0 + position) * p.out_stride + static_cast<size_t>(head) * D;
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
        const float x = __fdiv_rn(o[d], l);
        if constexpr (kBf16) {
            const __nv_bfloat16 b = __float2bfloat16(x);
            static_cast<__nv_bfloat16*>(p.out)[at + d * 32 + lane] = b;
            finite &= isfinite(__bfloat162float(b));
        } else {
            static_cast<float*>(p.out)[at + d * 32 + lane] = x;
            finite &= isfinite(x);
        }
    }
}

// One K/V head of a tile, a warp a row.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256) prompt_rows_kernel(PromptParams p) {
    pdl_wait();
    pdl_trigger();
    const int slot = static_cast<int>(kv8_div(blockIdx.x, p.by_heads)), kv_head = static_cast<int>(blockIdx.x - slot * p.by_heads.d);
    const PromptTile t = prompt_tile<256>(p, slot, blockIdx.x == gridDim.x - 1);
    if (t.index < 0) return;
    const int rows = min(p.tokens, t.length - t.first) * static_cast<int>(p.group.d);
    bool finite = true;
    for (int r = threadIdx.x >> 5; r < rows; r += 8) {
        const int at = static_cast<int>(kv8_div(r, p.group));
        prompt_row<D, kBf16>(p, t, t.first + at, kv_head * p.group.d + r - at * p.group.d, finite);
    }
    if (!__all_sync(kFull, finite) && (threadIdx.x & 31) == 0) prompt_flag(p, t.index, kStatusNonFinite);
}

}  // namespace phonon
