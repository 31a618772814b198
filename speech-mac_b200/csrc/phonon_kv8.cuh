// The 8-bit paged K/V cache (sm_100a): rows quantised as they are written,
// read back, and attended over.
//
// Format. A block is 16 positions of one K/V head; its keys and its values
// each share one scale 2^e with e the smallest integer in [kKv8MinExp,
// kKv8MaxExp] for which |x| <= 127 * 2^e over the block, and an element is
// held as the integer nearest x / 2^e, at most 127 in magnitude, plus 128.
// The scale is a power of two so that quantising, raising the scale of a
// partly filled block (the held integers divided by a power of two and
// rounded again) and reading back are exact but for the one rounding each
// names, in any order of operations; it costs at most one of the eight bits
// against a free scale. A block that fills position by position is rounded
// again only when its maximum crosses a power of two: the roundings' errors
// (1/2 unit of each scale, each scale at least twice the one before) sum to
// less than one unit of the last scale.
//
// Layout. pool: [layer][page][head][keys 16*D | values 16*D] bytes, exponents
// [layer][page][head][2], e + 127 in a byte. Keys lie [position][dim]. Values lie in the order in
// which the attention's lanes hold them: the 16 bytes of lane 4g + t in chunk
// j are dims 32j + 4g + w (w = byte / 4) of positions 2t, 2t + 1, 2t + 8,
// 2t + 9, so that a lane's 16-byte loads of either are matrix fragments as
// they stand: no shared memory, no transposition between the cache and the
// tensor cores.
#pragma once

#include "phonon_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace phonon {

constexpr int kKv8Block = kPage;  // positions that share a scale (a page)
constexpr int kKv8MinExp = -48, kKv8MaxExp = 64;
constexpr int kStatusInvalid = 1;   // PHONON_CUDA_INVALID_ARGUMENT
constexpr int kStatusCapacity = 5;  // PHONON_CUDA_CAPACITY

// One layer of a cache.
struct Kv8View {
    uint8_t* pool;
    uint8_t* exps;
    int pool_pages;
    int heads;  // K/V heads
};

// The sequences of a call. Sequence i holds lengths[i] + length_bias
// positions, the last of which are its rows [row_begin[i], row_begin[i + 1])
// of the call (rows_per_seq each where row_begin is null); position p lies in
// page pages[slot * page_stride + p / 16], slot = slots ? slots[i] : i.
struct Kv8Seqs {
    int n, rows, rows_per_seq;
    const int32_t* row_begin;
    const int32_t* lengths;
    int length_bias;
    const int32_t* slots;
    const int32_t* pages;
    int page_stride;
    int max_rows, max_length;
    int32_t* status;  // [n] or null
};

// The largest code wins: a sequence's status is set by many warps.
__device__ __forceinline__ void kv8_flag(const Kv8Seqs& s, int i, int code) {
    if (s.status) atomicMax(s.status + i, code);
}

struct Kv8Seq {
    int row0, count, length;
    const int32_t* pages;
};

// Sequence i's extent, checked against what the host launched for: rows
// outside the call's are refused (no row), lengths past the page table's or
// the launch's bound count as empty.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Seqs& s, int i) {
    Kv8Seq q;
    const int b = s.row_begin ? s.row_begin[i] : i * s.rows_per_seq;
    const int e = s.row_begin ? s.row_begin[i + 1] : b + s.rows_per_seq;
    q.length = s.lengths[i] + s.length_bias;
    q.row0 = b;
    q.count = e - b;
    if (b < 0 || e < b || e > s.rows || e - b > s.max_rows) {
        kv8_flag(s, i, kStatusInvalid);
        q.row0 = q.count = 0;
    }
    if (q.length < 0 || q.length > s.max_length) {
        kv8_flag(s, i, kStatusCapacity);
        q.length = 0;
    }
    q.pages = s.pages + static_cast<long long>(s.slots ? s.slots[i] : i) * s.page_stride;
    return q;
}

template <int D>
__device__ __forceinline__ uint8_t* kv8_block(const Kv8View& c, int page, int head, int which) {
    return c.pool + (static_cast<size_t>(page) * c.heads + head) * (2 * kKv8Block * D) + which * (kKv8Block * D);
}

__device__ __forceinline__ uint8_t* kv8_exp(const Kv8View& c, int page, int head) {
    return c.exps + (static_cast<size_t>(page) * c.heads + head) * 2;
}

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]

// The smallest e with amax <= 127 * 2^e, 127 = 1.984375 * 2^6.
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return min(max(e, kKv8MinExp), kKv8MaxExp);
}

// The nearest integer to x / 2^e (ties to even) plus 128 in the low byte:
// adding 1.5 * 2^23 + 128 rounds the exact quotient to an integer. |x| <= 127
// * 2^e.
__device__ __forceinline__ uint32_t kv8_code(float x, float inverse) {
    return __float_as_uint(__fmaf_rn(x, inverse, 12583040.0f));
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t kv8_pack(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Four held bytes of a scale 2^k times smaller (shrink = 2^-k) in the new one.
__device__ __forceinline__ uint32_t kv8_shrink(uint32_t w, float shrink) {
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = kv8_code(static_cast<float>(static_cast<int>((w >> (8 * k)) & 0xffu) - 128), shrink);
    return kv8_pack(r[0], r[1], r[2], r[3]);
}

// (Plain loads here and below, of all that a caller passes: these kernels start
// before the launch ahead of them has ended, which may still be writing it, and
// the read-only path takes its data for constant from a grid's start on.)
template <bool kBf16>
__device__ __forceinline__ float4 load_row4(const void* base, size_t at) {
    if constexpr (kBf16) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    } else {
        return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    }
}

template <bool kBf16>
__device__ __forceinline__ void store_row4(void* base, size_t at, float4 v) {
    if constexpr (kBf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = v;
    }
}

// ------------------------------------------------------------------- append
// n / d and n % d of a launch's block index for a d that the host knows:
// multiply and shift (Granlund and Montgomery's division by invariants, for
// n < 2^31, where the multiplier fits 32 bits).
struct Kv8Div {
    uint32_t d, mul, shift;
};

__device__ __forceinline__ uint32_t kv8_div(uint32_t n, Kv8Div d) { return d.d == 1 ? n : __umulhi(n, d.mul) >> d.shift; }

struct Kv8AppendParams {
    Kv8View cache;
    Kv8Seqs seqs;
    const void* rows[2];  // keys, values: [rows][heads][D], rows `stride` elements apart
    long long stride;
    int blocks;  // blocks of a sequence that its rows can touch, at most
    Kv8Div by_heads, by_blocks;
};

// Position of lane 4g + t's k-th byte of a value word (the layout above).
__device__ __forceinline__ int kv8_value_pos(int t, int k) { return 2 * t + (k & 1) + 8 * (k >> 1); }

// The values to quantise: non-finite ones count as 0, and none exceeds the
// largest that can be held.
__device__ __forceinline__ float4 kv8_sane(float4 v) {
    constexpr float kMost = 127.0f * 18446744073709551616.0f;  // 127 * 2^kKv8MaxExp
    float* f = &v.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = isfinite(f[k]) ? fminf(fmaxf(f[k], -kMost), kMost) : 0.0f;
    return v;
}

__device__ __forceinline__ float kv8_amax(float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }

// Above this the values are looked at one by one (kv8_sane).
constexpr float kKv8Tame = 1e20f;

// One warp writes one block's keys (which = 0) or values (1): the new rows'
// maximum, the scale, then the integers. A block's bytes are all owned by one
// warp; a partly filled block is read again only where its scale rises or a
// value word mixes old and new positions. Lane layout: keys, 4 dims of a row
// a lane (4-byte stores, rows coalesced); values, the lane's own chunks.
//
// Bound by latency (length, page id, rows, then stores) until a call has tens
// of megabytes: 4000 bf16 rows of 8 x 128 from the middle of a block on, 16
// sequences, 25 MB: 7.9 us. A warp a block and not a CTA: nothing to wait for
// but the warp's own loads, which are all in flight at once.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) kv8_append_kernel(Kv8AppendParams p) {
    constexpr int kLanesPerRow = D / 4, kRowsPerPass = 32 / kLanesPerRow, kPasses = kKv8Block / kRowsPerPass;
    constexpr int kChunks = D / 32;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const uint32_t item = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int which = item & 1;
    const uint32_t rest = kv8_div(item >> 1, p.by_heads);
    const int head = static_cast<int>((item >> 1) - rest * p.by_heads.d);
    const int i = static_cast<int>(kv8_div(rest, p.by_blocks)), bi = static_cast<int>(rest - i * p.by_blocks.d);
    if (i >= p.seqs.n) return;
    const Kv8Seq q = kv8_seq(p.seqs, i);
    const int start = max(q.length - q.count, 0);  // rows before position 0 go nowhere
    const int row0 = q.row0 + q.count - q.length;  // row of position 0
    const int block = start / kKv8Block + bi;
    const int p0 = block * kKv8Block;
    if (p0 >= q.length || q.count == 0) return;
    const int page = q.pages[block];
    const int lo = max(start - p0, 0), hi = min(q.length - p0, kKv8Block);  // new slots [lo, hi), kept [0, lo)
    const void* src = p.rows[which];
    const int g = lane >> 2, t = lane & 3;

    float4 x[kPasses];  // keys: rows of the passes; values: positions k of chunk j at 4j + k
    float amax = 0.0f, clean = 0.0f;
#pragma unroll
    for (int a = 0; a < kPasses; ++a) {
        const int slot = which == 0 ? a * kRowsPerPass + lane / kLanesPerRow : kv8_value_pos(t, a & 3);
        const int dim = which == 0 ? (lane % kLanesPerRow) * 4 : 32 * (a >> 2) + 4 * g;
        x[a] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (slot >= lo && slot < hi)
            x[a] = load_row4<kBf16>(src, static_cast<size_t>(row0 + p0 + slot) * p.stride + head * D + dim);
    }
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.cache.pool_pages)) {
        if (lane == 0) kv8_flag(p.seqs, i, kStatusInvalid);
        return;
    }
    uint8_t* ep = kv8_exp(p.cache, page, head) + which;
    const int held = lo > 0 ? *ep - 127 : kKv8MinExp;
    uint8_t* dst = kv8_block<D>(p.cache, page, head, which);
#pragma unroll
    for (int a = 0; a < kPasses; ++a) {
        amax = fmaxf(amax, kv8_amax(x[a]));
        clean = fmaf(x[a].x, 0.0f, fmaf(x[a].y, 0.0f, fmaf(x[a].z, 0.0f, fmaf(x[a].w, 0.0f, clean))));  // NaN once a value is not finite
    }
    if (!__all_sync(kFull, amax < kKv8Tame && clean == 0.0f)) {
        if (!__all_sync(kFull, clean == 0.0f) && lane == 0) kv8_flag(p.seqs, i, kStatusNonFinite);
        amax = 0.0f;
#pragma unroll
        for (int a = 0; a < kPasses; ++a) {
            x[a] = kv8_sane(x[a]);
            amax = fmaxf(amax, kv8_amax(x[a]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, o));
    const int e = max(kv8_exponent(amax), held);
    const float inverse = pow2i(-e), shrink = pow2i(held - e);
    const bool raised = lo > 0 && e > held;
    if (lane == 0) *ep = static_cast<uint8_t>(e + 127);

    if (which == 0) {
#pragma unroll
        for (int a = 0; a < kPasses; ++a) {
            const int slot = a * kRowsPerPass + lane / kLanesPerRow;
            uint32_t* at = reinterpret_cast<uint32_t*>(dst + slot * D) + lane % kLanesPerRow;
            if (slot >= lo && slot < hi)
                *at = kv8_pack(kv8_code(x[a].x, inverse), kv8_code(x[a].y, inverse), kv8_code(x[a].z, inverse),
                               kv8_code(x[a].w, inverse));
        }
        if (raised)
            for (int slot = lane / kLanesPerRow; slot < lo; slot += kRowsPerPass) {
                uint32_t* at = reinterpret_cast<uint32_t*>(dst + slot * D) + lane % kLanesPerRow;
                *at = kv8_shrink(*at, shrink);
            }
    } else {
        uint32_t fresh = 0;  // the new positions' bytes of a word
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int slot = kv8_value_pos(t, k);
            if (slot >= lo && slot < hi) fresh |= 0xffu << (8 * k);
        }
        if (fresh == 0 && !raised) return;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            uint4* at = reinterpret_cast<uint4*>(dst + j * 512) + lane;
            uint4 old = make_uint4(0, 0, 0, 0);
            if (fresh != 0xffffffffu) old = *at;
            uint32_t* w = &old.x;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const float* f[4] = {&x[4 * j].x, &x[4 * j + 1].x, &x[4 * j + 2].x, &x[4 * j + 3].x};
                const uint32_t mine = kv8_pack(kv8_code(f[0][d], inverse), kv8_code(f[1][d], inverse),
                                               kv8_code(f[2][d], inverse), kv8_code(f[3][d], inverse));
                // (bytes of positions behind the rows are shrunk too: they hold nothing)
                if (raised) w[d] = kv8_shrink(w[d], shrink);
                w[d] = (mine & fresh) | (w[d] & ~fresh);
            }
            *at = old;
        }
    }
}

// One new row a sequence (a decode step): D / 4 lanes per (sequence, head, keys
// or values), 4 dims a lane; nothing of the block is read unless the scale
// rises. 512 rows of 8 x 64 in fp32, 2 MB: 4.1 us, launch and three loads one
// after another (a warp a block, as above, takes 12.5).
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) kv8_append_one_kernel(Kv8AppendParams p) {
    constexpr int kLanes = D / 4;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, l = lane % kLanes;
    const uint32_t item = (blockIdx.x * blockDim.x + threadIdx.x) / kLanes;
    const int which = item & 1;
    const uint32_t rest = kv8_div(item >> 1, p.by_heads);
    const int head = static_cast<int>((item >> 1) - rest * p.by_heads.d), i = static_cast<int>(min(rest, p.seqs.n - 1u));
    const Kv8Seq q = kv8_seq(p.seqs, i);
    const bool real = rest < static_cast<uint32_t>(p.seqs.n) && q.count == 1 && q.length > 0;
    const int position = max(q.length - 1, 0), slot = position % kKv8Block;
    int page = -1;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (real) {
        page = q.pages[position / kKv8Block];
        x = load_row4<kBf16>(p.rows[which], static_cast<size_t>(q.row0) * p.stride + head * D + 4 * l);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.cache.pool_pages)) {
            if (l == 0) kv8_flag(p.seqs, i, kStatusInvalid);
            page = -1;
        }
    }
    uint8_t* ep = kv8_exp(p.cache, max(page, 0), head) + which;
    const int held = page >= 0 && slot > 0 ? *ep - 127 : kKv8MinExp;
    float amax = kv8_amax(x);
    const bool finite = isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w);
    if (!finite && page >= 0) kv8_flag(p.seqs, i, kStatusNonFinite);
    if (!finite || amax >= kKv8Tame) {
        x = kv8_sane(x);
        amax = kv8_amax(x);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, o));
    if (page < 0) return;
    const int e = max(kv8_exponent(amax), held);
    const float inverse = pow2i(-e), shrink = pow2i(held - e);
    if (l == 0) *ep = static_cast<uint8_t>(e + 127);
    const uint32_t c[4] = {kv8_code(x.x, inverse), kv8_code(x.y, inverse), kv8_code(x.z, inverse), kv8_code(x.w, inverse)};
    uint8_t* dst = kv8_block<D>(p.cache, page, head, which);
    if (which == 0) {
        uint32_t* at = reinterpret_cast<uint32_t*>(dst) + l;
        if (slot > 0 && e > held)
            for (int s = 0; s < slot; ++s) at[s * (D / 4)] = kv8_shrink(at[s * (D / 4)], shrink);
        at[slot * (D / 4)] = kv8_pack(c[0], c[1], c[2], c[3]);
    } else {
        // dims 4l.. are chunk l / 8, lanes 4 (l % 8) + t: four words of each t
        uint8_t* words = dst + (l >> 3) * 512 + (l & 7) * 64;
        if (slot > 0 && e > held)
            for (int w = 0; w < 16; ++w) {
                uint32_t* at = reinterpret_cast<uint32_t*>(words) + w;
                *at = kv8_shrink(*at, shrink);
            }
        const int t = (slot & 7) >> 1, k = (slot & 1) + 2 * (slot >> 3);
#pragma unroll
        for (int d = 0; d < 4; ++d) words[t * 16 + d * 4 + k] = static_cast<uint8_t>(c[d]);
    }
}

// ------------------------------------------- pages of a decode context (8 x 64)
// Where a block holds dim `dim` of position `slot` of its page.
template <int D>
__device__ __forceinline__ int kv8_byte(int which, int slot, int dim) {
    if (which == 0) return slot * D + dim;
    const int t = (slot & 7) >> 1, k = (slot & 1) + 2 * (slot >> 3);
    return (dim >> 5) * 512 + (((dim & 31) >> 2) * 4 + t) * 16 + (dim & 3) * 4 + k;
}

// Pages that a stream has just received (the step's (slot, index, page)
// updates) forget their scales in every layer: a stream may write its first
// row of a page at any slot.
__global__ void kv8_reset_kernel(uint8_t* exps, int layers, int pool_pages, int heads, const int32_t* updates, int n) {
    const int bytes = heads * 2;
    const long long total = static_cast<long long>(n) * layers * bytes;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int b = static_cast<int>(i % bytes), layer = static_cast<int>(i / bytes % layers);
        const int page = updates[3 * (i / bytes / layers) + 2];
        exps[(static_cast<size_t>(layer) * pool_pages + page) * bytes + b] = kKv8MinExp + 127;
    }
}

// kv_fill_kernel's values in 8 bits: below 2.449 in magnitude, so every block
// has the scale 2^-5.
__global__ void kv8_fill_kernel(uint8_t* pool, uint8_t* exps, int pool_pages, const int32_t* table, int n_layers, int length,
                                uint64_t seed) {
    constexpr int kBlockBytes = kKv8Block * kHeadDim;
    const long long per_pos = static_cast<long long>(n_layers) * 2 * kWidth;
    const long long total = per_pos * length;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int position = static_cast<int>(i / per_pos);
        const long long r = i % per_pos;
        const int layer = static_cast<int>(r / (2 * kWidth));
        const int which = static_cast<int>((r / kWidth) & 1);
        const int d = static_cast<int>(r % kWidth);
        const uint32_t h = hash32(seed * 0x9E3779B97F4A7C15ull + static_cast<uint64_t>(i));
        const float u = (static_cast<float>(h & 0xffff) + static_cast<float>(h >> 16)) * (1.0f / 65536.0f);
        const float v = (u - 1.0f) * 2.449f;
        const size_t block = (static_cast<size_t>(layer) * pool_pages + table[position / kPage]) * kHeads + (d >> 6);
        pool[(block * 2 + which) * kBlockBytes + kv8_byte<kHeadDim>(which, position % kPage, d & 63)] =
            static_cast<uint8_t>(kv8_code(v, 32.0f));
        if ((d & 63) == 0 && position % kPage == 0) exps[block * 2 + which] = 127 - 5;
    }
}

// --------------------------------------------------------------------- read
// (held integer) * 2^e. Bound by the bytes: 110 sequences of up to 2048
// positions, 8 heads of 128, to bf16: 69.5 us, 6.0 TB/s, 92 % of the copy rate
// (124 with the bytes of a block taken one at a time); one sequence of 8000, 8 x
// 64, to fp32, 41 MB: 10.2 us, of which 4 are launch and latency.
struct Kv8ReadParams {
    Kv8View cache;
    Kv8Seqs seqs;
    void* rows[2];
    long long stride;
    int blocks;
};

// One warp reads one block's keys or values back: held byte - 128 times 2^e,
// exact in fp32. Rows of positions before 0, of empty and of bad pages are 0.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) kv8_read_kernel(Kv8ReadParams p) {
    constexpr int kLanesPerRow = D / 4, kRowsPerPass = 32 / kLanesPerRow, kPasses = kKv8Block / kRowsPerPass;
    constexpr int kChunks = D / 32;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long item = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int which = static_cast<int>(item & 1);
    long long rest = item >> 1;
    const int head = static_cast<int>(rest % p.cache.heads);
    rest /= p.cache.heads;
    const int bi = static_cast<int>(rest % p.blocks);
    rest /= p.blocks;
    if (rest >= p.seqs.n) return;
    const int i = static_cast<int>(rest);
    const Kv8Seq q = kv8_seq(p.seqs, i);
    // positions [length - count, length), counted from the block of the first (negative ones included)
    const int start = q.length - q.count;
    const int block = (start >= 0 ? start / kKv8Block : -((kKv8Block - 1 - start) / kKv8Block)) + bi;
    const int p0 = block * kKv8Block;
    if (p0 >= q.length || q.count == 0) return;
    const int row0 = q.row0 - start;
    int page = block >= 0 ? q.pages[block] : -1;
    if (block >= 0 && static_cast<unsigned>(page) >= static_cast<unsigned>(p.cache.pool_pages)) {
        if (lane == 0) kv8_flag(p.seqs, i, kStatusInvalid);
        page = -1;
    }
    const int lo = max(start - p0, 0), hi = min(q.length - p0, kKv8Block);
    const uint8_t* src = page >= 0 ? kv8_block<D>(p.cache, page, head, which) : nullptr;
    const float unit = page >= 0 ? pow2i(kv8_exp(p.cache, page, head)[which] - 127) : 0.0f;
    void* dst = p.rows[which];
    auto value = [&](uint32_t w, int k) {
        return (static_cast<float>((w >> (8 * k)) & 0xffu) - 128.0f) * unit;
    };
    const int g = lane >> 2, t = lane & 3;
    if (which == 0) {
        uint32_t w[kPasses];
#pragma unroll
        for (int a = 0; a < kPasses; ++a) {
            const int slot = a * kRowsPerPass + lane / kLanesPerRow;
            w[a] = src && slot >= lo && slot < hi
                       ? *(reinterpret_cast<const uint32_t*>(src + slot * D) + lane % kLanesPerRow)
                       : 0x80808080u;
        }
#pragma unroll
        for (int a = 0; a < kPasses; ++a) {
            const int slot = a * kRowsPerPass + lane / kLanesPerRow;
            if (slot >= lo && slot < hi)
                store_row4<kBf16>(dst, static_cast<size_t>(row0 + p0 + slot) * p.stride + head * D + (lane % kLanesPerRow) * 4,
                                  make_float4(value(w[a], 0), value(w[a], 1), value(w[a], 2), value(w[a], 3)));
        }
    } else {
        uint4 w[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
            w[j] = src ? *(reinterpret_cast<const uint4*>(src + j * 512) + lane)
                       : make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int slot = kv8_value_pos(t, k);
                if (slot >= lo && slot < hi)
                    store_row4<kBf16>(dst, static_cast<size_t>(row0 + p0 + slot) * p.stride + head * D + 32 * j + 4 * g,
                                      make_float4(value(w[j].x, k), value(w[j].y, k), value(w[j].z, k), value(w[j].w, k)));
            }
    }
}

// ---------------------------------------------------------------- attention
// out[r] = sum_k softmax_k(scale q_r . K_k) V_k over the positions k that row
// r (at position p_r) sees: k <= p_r, and k > p_r - window where a window is
// set. Rows that see nothing get 0.
//
// Per block the tensor cores compute S^T = K q^T (16 positions x 8 columns)
// and O^T += V^T P^T (16 dims x 8 columns): the cache is the A operand, rows
// are columns, so that a decode step's single row (times the grouped heads)
// costs half the instructions that it would as M. A block's scales enter in
// fp32: with s = scale log2(e) 2^eK (q.K) + eV, the weight 2^(s - M) is the
// softmax weight times the block's value scale, so that O needs no scaling of
// its own, and the sum of weights takes 2^(s - M - eV). M is the running
// maximum of s.
//
// The weights are rounded to a step of the largest there can be (below), so
// eV is taken relative to a reference of the warp's pages: their largest that
// is at most kKv8Spread above their smallest. Blocks that do not lie within
// kKv8Spread below it (one loud position among quiet ones raises its block's
// scale by up to 2^112, whatever its weight) are multiplied in fp32, element
// by element, behind the others: a step of theirs would be all that the other
// blocks weigh, or the other way round. (512 sequences of about 1000 positions:
// 87 us, with one position in 1000 that is 2^20 times louder 103, in 100 142.)
//
// Up to four rows that share a head (a decode step): 8-bit integer products,
// the cache's bytes as they lie. q is held as an integer of 31 bits relative
// to the row's maximum (an element keeps fp32's 24 bits down to 2^-7 of it,
// bf16's 8 down to 2^-23), split into signed bytes: columns 2r, 2r + 1 are the
// first two of row r and a second column tile has the others. A score's sums
// are exact; so are those of the output per turn, with the weights as integers
// of 32 bits, a byte a column. (The cache's bytes are unsigned, 128 too large:
// products with a constant -128 in their place start the sums.) What is left
// are q's and the weights' own roundings (2^-32 of a row's largest; 2^-33 of
// the largest weight, or its fp32's) and the turns' fp32 sums.
//
// More rows: products of halves, the conversion of a block's bytes shared by
// the rows. Byte | 0x6400 is the half 1152 + integer, minus 1152 the integer,
// exactly, one byte permutation and one subtraction for two. The products are
// exact in the fp32 accumulators. fp32 rows: q (scaled by a power of two to a
// row maximum near 2^12) and the weights enter as two halves each, 22 bits.
// bf16 rows: q fits one half (8 bits), a weight is rounded to one half (11 bits,
// under the output's 8).
struct Kv8AttnParams {
    Kv8View cache;
    Kv8Seqs seqs;
    const void* q;
    void* out;
    long long q_stride, out_stride;  // elements between rows; a row is [heads][D]
    Kv8Div group;                    // query heads per K/V head
    float scale, scale_low;          // softmax scale times log2(e), and what its rounding left
    int window;                      // 0: none
    Kv8Div by_items, by_heads, by_tiles;  // (sequence, row tile, K/V head) items; K/V heads; row tiles of a sequence
    int splits;                            // of an item, at most
    int split_pages;                       // pages of a split
    int tile_rows;                         // rows of a row tile
    float* part;                     // [items * splits][rows of a tile][D]
    float4* part_ml;                 // [items * splits][rows of a tile]: M, sum, eV's reference
    unsigned* arrived;               // [items], zero between launches
};

constexpr float kKv8WeightBits = 14.0f;  // weights are held times 2^14: a half keeps 11 bits down to 2^-28

// The value scales 2^(ref - kKv8Spread) to 2^ref enter the weights; more would
// cost as many of the smallest scale's bits (byte products keep 2^-25 of the
// largest weight at the bottom of the range, halves 2^-31).
constexpr int kKv8Spread = 8;
constexpr int kKv8Above = 64;  // no block's scale is further above ref, so that sums stay inside fp32

// The reference of blocks with value scales (biased exponents) from lo to hi.
__device__ __forceinline__ int kv8_reference(int lo, int hi) { return max(min(hi, lo + kKv8Spread), hi - kKv8Above); }

// Whether a block's scale, relative to the reference, enters the weights.
__device__ __forceinline__ bool kv8_near(int ev) { return static_cast<unsigned>(ev + kKv8Spread) <= static_cast<unsigned>(kKv8Spread); }

// Byte k of a cache word as a number.
__device__ __forceinline__ float kv8_number(uint32_t w, int k) { return __uint_as_float(0x4b000000u | (w >> (8 * k) & 0xffu)) - 8388736.0f; }

// Weights as integers of 32 bits: 1 is the largest float below 2^32.
constexpr float kKv8FixedScale = 4294967040.0f;

enum Kv8Mode : int { KV8_HALF_BF16 = 0, KV8_HALF_F32 = 1, KV8_INT_BF16 = 2, KV8_INT_F32 = 3 };

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d = c + 16 x 32 bytes by 32 x 8 bytes; kKinds: "u8.s8", "u8.u8", "s8.s8" or
// "s8.u8".
#define KV8_IMMA(NAME, KINDS)                                                                                        \
    __device__ __forceinline__ void NAME(int (&d)[4], const int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,      \
                                         uint32_t a3, uint32_t b0, uint32_t b1) {                                    \
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." KINDS                                                  \
                     ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"                                \
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                \
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3])); \
    }
KV8_IMMA(imma_u8_s8, "u8.s8")
KV8_IMMA(imma_u8_u8, "u8.u8")
KV8_IMMA(imma_s8_s8, "s8.s8")
KV8_IMMA(imma_s8_u8, "s8.u8")
#undef KV8_IMMA
constexpr uint32_t kKv8Minus128 = 0x80808080u;  // four signed bytes

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 x, y, z, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 w, x, y, z; "
        "mov.b64 {%0, %1}, w;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// 2^x, results below 2^-126 are 0 (weights are at most 2^14).
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Bytes 0, 1 (kHigh: 2, 3) of a cache word as the halves byte - 128.
template <bool kHigh>
__device__ __forceinline__ uint32_t kv8_halves(uint32_t w) {
    uint32_t u = __byte_perm(w, 0x64646464u, kHigh ? 0x4342 : 0x4140);
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&u), bias);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 half2_floats(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

// M, sum of weights, reference of eV (biased) and four dims of a row, over some of its positions.
struct Kv8Share {
    float m, l;
    int ref;
    float4 a;
};

__device__ __forceinline__ Kv8Share kv8_nothing() { return {-INFINITY, 0.0f, 127, make_float4(0.0f, 0.0f, 0.0f, 0.0f)}; }

__device__ __forceinline__ void kv8_fold(Kv8Share& s, float4 ml, float4 b) {
    // the sums go into the larger reference (an exact power of two), then the larger maximum
    const int other = __float_as_int(ml.z);
    if (s.m == -INFINITY && !isnan(s.l)) s.ref = other;  // nothing yet: as it comes
    const int ref = ml.x == -INFINITY ? s.ref : max(s.ref, other);
    const float x = fmaxf(s.m, ml.x);
    const float wa = s.m == -INFINITY ? 0.0f : ex2(s.m - x), wb = ml.x == -INFINITY ? 0.0f : ex2(ml.x - x);
    const float oa = wa * pow2i(s.ref - ref), ob = wb * pow2i(min(other - ref, 0));
    s.m = x;
    s.ref = ref;
    s.l = s.l * wa + ml.y * wb;
    s.a = make_float4(s.a.x * oa + b.x * ob, s.a.y * oa + b.y * ob, s.a.z * oa + b.z * ob, s.a.w * oa + b.w * ob);
}

// Four dims of row rho of a K/V head's rows, to the output.
template <int D, bool kBf16>
__device__ __forceinline__ void kv8_store(const Kv8AttnParams& p, int row0, int rho, int head, int d, float4 v) {
    const int at = static_cast<int>(kv8_div(rho, p.group));
    store_row4<kBf16>(p.out, static_cast<size_t>(row0 + at) * p.out_stride + static_cast<size_t>(head * p.group.d + rho - at * p.group.d) * D + d, v);
}

// What turns a row's sums into its output; unit: what a weight of 1 is held as, inverted.
__device__ __forceinline__ float kv8_inverse(float l, int ref, float unit) {
    return l > 0.0f || isnan(l) ? __fdiv_rn(pow2i(ref - 127) * unit, l) : 0.0f;
}

// The end of a split item, after the CTA has written its shares to the
// scratch: the split that arrives last merges all of them, in their order, so
// that results do not depend on who arrives when. Threads 0 to kThreads - 1,
// whose barrier is sync; `scratch`: 2 * kThreads float4 of shared memory.
template <int D, bool kBf16, int kThreads, int kCells, typename Sync>
__device__ __forceinline__ void kv8_merge(const Kv8AttnParams& p, float unit, const Sync& sync, float4* scratch, int* s_last, uint32_t item,
                                          int active, int tile_rows, int n_rows, int row0, int rho0, int head) {
    constexpr int kQuads = D / 4;
    const size_t slot = static_cast<size_t>(item) * p.splits;
    const auto finish = [&](int cell, const Kv8Share& s) {
        const int d = cell % kQuads * 4;
        const float inv = kv8_inverse(s.l, s.ref, unit);
        kv8_store<D, kBf16>(p, row0, rho0 + cell / kQuads, head, d, make_float4(s.a.x * inv, s.a.y * inv, s.a.z * inv, s.a.w * inv));
    };
    sync();
    if (threadIdx.x == 0) {
        unsigned n;  // releases the CTA's partial results (ordered before by the barrier), acquires the others'
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(p.arrived + item) : "memory");
        *s_last = n + 1 == static_cast<unsigned>(active);
        if (*s_last) p.arrived[item] = 0;
    }
    sync();
    if (!*s_last) return;
    // Few rows: the threads share a row's splits, each every subs-th, and the
    // subs meet in shared memory; four splits of kCells cells (four dims of a
    // row) are loaded at a time.
    const int cells = n_rows * kQuads, subs = max(1, min(active, kThreads / cells));
    for (int x0 = threadIdx.x; x0 < cells * subs; x0 += kCells * kThreads) {
        Kv8Share s[kCells];
        int at[kCells], sub[kCells];
#pragma unroll
        for (int c = 0; c < kCells; ++c) {
            const int x = min(x0 + c * kThreads, cells * subs - 1);
            sub[c] = x / cells;
            at[c] = x - sub[c] * cells;
            s[c] = kv8_nothing();
        }
        for (int step = 0; step < active; step += 4 * subs) {
            float4 ml[kCells][4], a[kCells][4];
#pragma unroll
            for (int c = 0; c < kCells; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const size_t at_part = (slot + min(step + sub[c] + k * subs, active - 1)) * tile_rows + at[c] / kQuads;
                    ml[c][k] = __ldcg(p.part_ml + at_part);
                    a[c][k] = __ldcg(reinterpret_cast<const float4*>(p.part + at_part * D + at[c] % kQuads * 4));
                }
#pragma unroll
            for (int c = 0; c < kCells; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (step + sub[c] + k * subs < active) kv8_fold(s[c], ml[c][k], a[c][k]);
        }
#pragma unroll
        for (int c = 0; c < kCells; ++c) {
            const int x = x0 + c * kThreads;
            if (x >= cells * subs) break;
            if (subs == 1) {
                finish(at[c], s[c]);
            } else {
                scratch[x] = s[c].a;
                scratch[cells * subs + x] = make_float4(s[c].m, s[c].l, __int_as_float(s[c].ref), 0.0f);
            }
        }
    }
    if (subs == 1) return;
    sync();
    for (int cell = threadIdx.x; cell < cells; cell += kThreads) {
        Kv8Share s = kv8_nothing();
        for (int sub = 0; sub < subs; ++sub) kv8_fold(s, scratch[cells * subs + sub * cells + cell], scratch[sub * cells + cell]);
        finish(cell, s);
    }
}

// A lane's share of a block: its keys are D/4 dims of positions g, g + 8 (the
// t-th 16 bytes of each 64; 8 of 32 where D is 32), its values D/32 chunks of
// 16 bytes. The lane copies them into its warp's ring in shared memory and
// reads them back itself, so no other thread is waited for: 16 bytes of lane
// 0, of lane 1, ... per chunk, without bank conflicts.
// (0 of `bytes` read: zeros are written and the source is not touched)
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copy8(uint32_t dst, const uint8_t* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes / 2) : "memory");
}

template <int D>
__device__ __forceinline__ void kv8_copy(uint32_t dst, const uint8_t* block, int lane, int bytes) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (D == 32) {
            copy8(dst + h * 256 + lane * 8, block + (g + 8 * h) * D + t * 8, bytes);
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
                copy16(dst + (h * (D / 64) + c) * 512 + lane * 16, block + (g + 8 * h) * D + c * 64 + t * 16, bytes);
        }
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
        copy16(dst + kKv8Block * D + j * 512 + lane * 16, block + kKv8Block * D + j * 512 + lane * 16, bytes);
}

// Key words [position g, g + 8][4 dims each], value words [2 x 16-dim tiles].
template <int D>
__device__ __forceinline__ void kv8_key_words(uint32_t (&w)[2][D / 16], const uint8_t* page, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (D == 32) {
            const uint2 v = *reinterpret_cast<const uint2*>(page + h * 256 + lane * 8);
            w[h][0] = v.x;
            w[h][1] = v.y;
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const uint4 v = *reinterpret_cast<const uint4*>(page + (h * (D / 64) + c) * 512 + lane * 16);
                w[h][4 * c] = v.x;
                w[h][4 * c + 1] = v.y;
                w[h][4 * c + 2] = v.z;
                w[h][4 * c + 3] = v.w;
            }
        }
    }
}

// The first dim of key word c.
template <int D>
__device__ __forceinline__ int kv8_key_dim(int t, int c) {
    return D == 32 ? t * 8 + c * 4 : (c >> 2) * 64 + t * 16 + (c & 3) * 4;
}

// One CTA: one (sequence, row tile, K/V head, split). Its warps take the
// split's pages PB at a time in turn, each with an online softmax of its own,
// and meet in shared memory; the last split to arrive merges them in order.
// Pages come by asynchronous copies, kStages - 1 turns ahead, in a ring that a
// warp has to itself: the copies, not registers, hold what is in flight, which
// leaves room for 12 to 16 warps an SM (24 and more in single-warp CTAs). Page
// ids and scales are fetched a lane each, 32 / PB turns at a time.
//
// Decode steps are bound by the cache's bytes: 512 sequences of up to 2048
// positions, 8 x 64, 526 MB, 87.7 us (6.0 TB/s, 93 % of the copy rate); as halves
// with register loads 137, with the ring 101, as bytes 95. 48 of up to 4096, 32
// heads on 8 x 128, 225 MB, 49 us: a CTA's start and end (4 us) against 30 us of
// pages, three CTAs an SM. 8 of 8000: 18 us, 5.7 of them the chain of loads
// before the first page and 3 the merge. One of 1000: 6.5 us, all latency. 64 x
// 16 rows over 250 keys 14.0 us, 4 chunks of up to 256 rows 27.3 us: bound by
// the halves' matrix rate (2.1 clocks an m16n8k16 on an SM, two of them in
// fp32) and, in bf16 with 128 dims, by the conversion of the bytes.
// A persistent form that cut the positions of all items into equal lines for
// the resident CTAs: 99 us and 26 (8 of 8000), since each cut costs a merge.
template <int D, int NT, int PB, int kStages, int kMode, int kWarps, int kCtas>
__global__ void __launch_bounds__(32 * kWarps, kCtas) kv8_attention_kernel(Kv8AttnParams p) {
    constexpr bool kBf16 = kMode == KV8_HALF_BF16 || kMode == KV8_INT_BF16, kFine = kMode == KV8_HALF_F32;
    constexpr bool kInt = kMode == KV8_INT_BF16 || kMode == KV8_INT_F32;
    static_assert(!kInt || (NT == 1 && PB % 2 == 0), "four rows, values multiplied two pages at a time");
    constexpr int kRows = kInt ? 4 : 8 * NT;
    constexpr int RT = kInt ? 1 : 2;  // rows of a column tile that a lane holds scores of
    constexpr int KS = D / 16;         // 16-dim steps of a score, and 16-dim tiles of an output
    constexpr int kTurns = 32 / PB, kPageBytes = 2 * kKv8Block * D;
    extern __shared__ __align__(16) uint8_t s_ring[];  // [kWarps][kStages][PB][kPageBytes], then the warps' results
    float(*s_o)[kRows][D] = reinterpret_cast<float(*)[kRows][D]>(s_ring);
    __shared__ float4 s_ml[kWarps][kRows];  // M, sum, eV's reference
    __shared__ int s_last, s_lowest[kWarps];
    __shared__ int4 s_range[kWarps];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // block index: heads fastest (a page's heads are neighbours), then row
    // tiles, sequences and, last to first, splits: the splits that only long
    // sequences have start first, the short sequences' work ends the launch
    const uint32_t later = kv8_div(blockIdx.x, p.by_items), item = blockIdx.x - later * p.by_items.d;
    const uint32_t entry = kv8_div(item, p.by_heads);
    const int head = static_cast<int>(item - entry * p.by_heads.d);
    const int split = p.splits - 1 - static_cast<int>(later);
    const int i = static_cast<int>(kv8_div(entry, p.by_tiles));
    const int tile = static_cast<int>(entry - i * p.by_tiles.d);
    const Kv8Seq sq = kv8_seq(p.seqs, i);
    const int rows = sq.count * static_cast<int>(p.group.d) - tile * kRows;  // rows left from this tile on
    if (rows <= 0) return;
    const int n_rows = min(rows, kRows), rho0 = tile * kRows;
    const int at0 = sq.length - sq.count;  // position of the sequence's first row
    auto token = [&](int rho) { return static_cast<int>(kv8_div(rho, p.group)); };
    const int pos_lo = at0 + token(rho0), pos_hi = at0 + token(rho0 + n_rows - 1);
    const int key_end = min(pos_hi + 1, sq.length);
    const int page_begin = p.window ? max(pos_lo - p.window + 1, 0) / kKv8Block : 0;
    const int pages = key_end > 0 ? (key_end + kKv8Block - 1) / kKv8Block - page_begin : 0;
    const int active = max(1, min(p.splits, (pages + p.split_pages - 1) / p.split_pages));
    if (split >= active) return;
    const int per = (pages + active - 1) / active;
    const int first = page_begin + min(pages, split * per), last = page_begin + min(pages, (split + 1) * per);
    // pages that every row of the tile sees whole: [whole_first, whole_last)
    const int whole_last = max(pos_lo + 1, 0) / kKv8Block;
    const int whole_first = p.window && pos_hi >= p.window ? (pos_hi - p.window) / kKv8Block + 1 : 0;

    // this lane's page of kTurns turns of the warp, and of the kTurns after them: its id (-1: none) and scales
    constexpr int kStep = kWarps * PB;
    const int own = first + warp * PB + lane / PB * kStep + lane % PB;
    const uint8_t* exps = p.cache.exps + head * 2;
    int ids[2], scales[2];
    auto fetch = [&](int half, int turn) {
        const int at = own + turn * kStep;
        ids[half] = at < last ? sq.pages[at] : -1;
        if (at < last && static_cast<unsigned>(ids[half]) >= static_cast<unsigned>(p.cache.pool_pages)) {
            kv8_flag(p.seqs, i, kStatusInvalid);
            ids[half] = -1;  // its positions are not seen
        }
        scales[half] = ids[half] >= 0
                           ? *reinterpret_cast<const unsigned short*>(exps + static_cast<size_t>(ids[half]) * p.cache.heads * 2)
                           : 127 | 127 << 8;
    };
    const uint8_t* base = p.cache.pool + static_cast<size_t>(head) * kPageBytes;
    const size_t page_bytes = static_cast<size_t>(p.cache.heads) * kPageBytes;
    const uint8_t* ring = s_ring + warp * (kStages * PB * kPageBytes);
    const uint32_t ring_addr = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    auto copy = [&](int half, int turn, int stage) {  // turn's pages into the stage; always one group
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            const int id = __shfl_sync(kFull, ids[half], turn % kTurns * PB + b);
            kv8_copy<D>(ring_addr + (stage * PB + b) * kPageBytes, base + max(id, 0) * page_bytes, lane, id >= 0 ? 16 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the rows of q on their way before the page ids are waited for
    float4 q[NT][KS];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int rho = rho0 + min(kInt ? g >> 1 : n * 8 + g, n_rows - 1), at = token(rho);
        const size_t row = static_cast<size_t>(sq.row0 + at) * p.q_stride +
                           static_cast<size_t>(head * p.group.d + rho - at * p.group.d) * D;
#pragma unroll
        for (int c = 0; c < KS; ++c) q[n][c] = load_row4<kBf16>(p.q, row + kv8_key_dim<D>(t, c));
    }
    fetch(0, 0);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) copy(0, s, s);
    fetch(1, kTurns);
    // q as B fragments; column g is row g (halves), or byte g % 2 of row g / 2 (qh) and byte 2 + g % 2 (ql)
    constexpr int QS = kInt ? D / 32 : KS;  // steps of a score
    uint32_t qh[NT][QS][2], ql[NT][kFine || kInt ? QS : 1][2];
    float f[NT][RT];  // 2^(row exponent) of the lane's rows
    int pos[NT][RT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = kInt ? g >> 1 : n * 8 + g;
        const float4(&v)[KS] = q[n];
        float amax = 0.0f;
        bool finite = true;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            finite &= isfinite(v[c].x) & isfinite(v[c].y) & isfinite(v[c].z) & isfinite(v[c].w);
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v[c].x), fabsf(v[c].y)), fmaxf(fabsf(v[c].z), fabsf(v[c].w))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
        const unsigned bad = __ballot_sync(kFull, !finite);
        const bool row_bad = (bad >> (lane & ~3) & 0xfu) != 0;
        if (row_bad && t == 0 && r < n_rows) kv8_flag(p.seqs, i, kStatusNonFinite);
        // exponent of the maximum, kept where both powers below are normal
        // (integers: the maximum times 2^(kTop - e) is at most 1.984375 * 2^kTop, whose bytes fit)
        constexpr int kTop = kInt ? 30 : 12;
        const uint32_t top_bits = __float_as_uint(amax);
        const int above = kInt && (top_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0;
        const int e = min(max(static_cast<int>(top_bits >> 23) - 127 + above, kTop - 126), 126);
        const float up = pow2i(kTop - e), back = pow2i(e - kTop);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const float x[4] = {v[c].x * up, v[c].y * up, v[c].z * up, v[c].w * up};
            if constexpr (kInt) {
                // signed bytes ((d0 * 256 + d1) * 256 + d2) * 256 + d3, |d0| <= 127 (unsigned: a row that is not finite wraps)
                uint32_t first = 0, rest = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t y3 = static_cast<uint32_t>(__float2int_rn(x[k]));
                    const int y2 = static_cast<int>(y3 + 128) >> 8, y1 = (y2 + 128) >> 8, y0 = (y1 + 128) >> 8;
                    first |= (static_cast<uint32_t>(g & 1 ? y1 : y0) & 0xffu) << (8 * k);
                    rest |= ((g & 1 ? y3 : static_cast<uint32_t>(y2)) & 0xffu) << (8 * k);
                }
                qh[n][c / 2][c % 2] = first;
                ql[n][c / 2][c % 2] = rest;
            } else {
                qh[n][c][0] = half2_bits(x[0], x[1]);
                qh[n][c][1] = half2_bits(x[2], x[3]);
                if constexpr (kFine) {
                    const float2 h0 = half2_floats(qh[n][c][0]), h1 = half2_floats(qh[n][c][1]);
                    ql[n][c][0] = half2_bits(x[0] - h0.x, x[1] - h0.y);
                    ql[n][c][1] = half2_bits(x[2] - h1.x, x[3] - h1.y);
                }
            }
        }
        const float fr = row_bad ? __int_as_float(0x7fc00000) : back;  // a bad row's output is NaN
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            f[n][k] = __shfl_sync(kFull, fr, 8 * t + 4 * k);
            const int lane_row = kInt ? t : n * 8 + 2 * t + k;
            pos[n][k] = at0 + token(rho0 + min(lane_row, n_rows - 1));
        }
    }

    // what a score's sums start from: -128 times those of q's bytes
    int q_base[4] = {0, 0, 0, 0}, q_base2[4] = {0, 0, 0, 0};
    if constexpr (kInt) {
#pragma unroll
        for (int c = 0; c < QS; ++c) {
            imma_s8_s8(q_base, q_base, kKv8Minus128, kKv8Minus128, kKv8Minus128, kKv8Minus128, qh[0][c][0], qh[0][c][1]);
            imma_s8_s8(q_base2, q_base2, kKv8Minus128, kKv8Minus128, kKv8Minus128, kKv8Minus128, ql[0][c][0], ql[0][c][1]);
        }
    }

    // O: [16-dim tile][column tile][accumulators] (halves), or the lane's row of dims g, g + 8 of a tile
    constexpr int OT = kInt ? 2 : 4;
    float o[KS][NT][OT], m[NT][RT], l[NT][RT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            m[n][k] = -INFINITY;
            l[n][k] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < OT; ++j) o[k][n][j] = 0.0f;
    }
    const int from0 = 8 * t + (g >> 1), from1 = from0 + 4;   // lanes with the weights of positions 2t, 2t + 1 of row g / 2
    const uint32_t pick = g & 1 ? 0x6240u : 0x7351u;         // the weight byte that column g multiplies

    // value scales, biased: the smallest of the CTA's first pages and of the warp's so far, the warp's largest up to
    // kKv8Spread above it, the largest of all, and whether a page is hidden (kept out of the registers between windows)
    const int lowest = __reduce_min_sync(kFull, ids[0] >= 0 ? scales[0] >> 8 : 255);
    if (lane == 0) s_lowest[warp] = lowest;
    if constexpr (kWarps > 1) __syncthreads();
    else __syncwarp();
    const auto start = [&] {
        int lo = 255;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) lo = min(lo, s_lowest[w]);
        return make_int4(lo, 0, 0, 0);
    };
    int ref = 127;  // what eV is relative to
    // Takes a window's pages into the range and hides those whose value scale does not enter the weights: the lane's, or -1.
    const auto look = [&](int4& range) {
        const int ev = ids[0] >= 0 ? scales[0] >> 8 : 255;
        range.x = min(range.x, __reduce_min_sync(kFull, ev));
        range.y = max(range.y, __reduce_max_sync(kFull, ev <= range.x + kKv8Spread && ev < 255 ? ev : 0));
        range.z = max(range.z, __reduce_max_sync(kFull, ev < 255 ? ev : 0));
        if (range.z) ref = max(range.y ? min(range.y, range.x + kKv8Spread) : range.x, range.z - kKv8Above);
        const int hidden = ids[0] >= 0 && !kv8_near(ev - ref) ? ids[0] : -1;
        if (hidden >= 0) ids[0] = -1;
        range.w |= __any_sync(kFull, hidden >= 0);
        return hidden;
    };
    {
        int4 range = start();
        look(range);
        if (lane == 0) s_range[warp] = range;
    }
    int turn = 0, stage = 0;
    for (int at = first + warp * PB; at < last; at += kStep, ++turn, stage = stage + 1 == kStages ? 0 : stage + 1) {
        if (turn && turn % kTurns == 0) {
            ids[0] = ids[1];
            scales[0] = scales[1];
            fetch(1, turn + kTurns);
            const int before = ref;
            __syncwarp();
            int4 range = s_range[warp];
            look(range);
            __syncwarp();
            if (lane == 0) s_range[warp] = range;
            if (ref != before) {  // O in the new unit: an exact power of two
                const float by = pow2i(before - ref);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < OT; ++j) o[k][n][j] *= by;
            }
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        {
            const int ahead = turn + kStages - 1, slot = stage == 0 ? kStages - 1 : stage - 1;
            if (turn % kTurns + kStages - 1 < kTurns) copy(0, ahead, slot);
            else copy(1, ahead, slot);
        }
        const uint8_t* pages_at = ring + stage * (PB * kPageBytes);
        int id[PB], ex[PB];
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            id[b] = __shfl_sync(kFull, ids[0], turn % kTurns * PB + b);
            ex[b] = __shfl_sync(kFull, scales[0], turn % kTurns * PB + b);
        }
        float s[PB][NT][2][RT];  // s + eV of positions g, g + 8
        float less[PB];          // 2^-eV
#pragma unroll
        for (int b = 0; b < PB; ++b) {
            float c4[NT][4];  // q.K: positions g, g + 8 of the lane's rows
            uint32_t kw[2][D / 16];
            kv8_key_words<D>(kw, pages_at + b * kPageBytes, lane);
            if constexpr (kInt) {
                int x[4], y[4];
#pragma unroll
                for (int c = 0; c < QS; ++c) {
                    imma_u8_s8(x, c ? x : q_base, kw[0][2 * c], kw[1][2 * c], kw[0][2 * c + 1], kw[1][2 * c + 1], qh[0][c][0], qh[0][c][1]);
                    imma_u8_s8(y, c ? y : q_base2, kw[0][2 * c], kw[1][2 * c], kw[0][2 * c + 1], kw[1][2 * c + 1], ql[0][c][0], ql[0][c][1]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    c4[0][2 * h] = fmaf(static_cast<float>(x[2 * h] * 256 + x[2 * h + 1]), 65536.0f,
                                        static_cast<float>(y[2 * h] * 256 + y[2 * h + 1]));
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n) c4[n][0] = c4[n][1] = c4[n][2] = c4[n][3] = 0.0f;
#pragma unroll
                for (int c = 0; c < KS; ++c) {
                    const uint32_t wa = kw[0][c], wb = kw[1][c];
                    const uint32_t a0 = kv8_halves<false>(wa), a1 = kv8_halves<false>(wb);
                    const uint32_t a2 = kv8_halves<true>(wa), a3 = kv8_halves<true>(wb);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816(c4[n], a0, a1, a2, a3, qh[n][c][0], qh[n][c][1]);
                        if constexpr (kFine) mma16816(c4[n], a0, a1, a2, a3, ql[n][c][0], ql[n][c][1]);
                    }
                }
            }
            const float uk = __int_as_float((ex[b] & 0xff) << 23);
            const int ev = (ex[b] >> 8) - ref;
            const float add = static_cast<float>(ev);
            less[b] = pow2i(-ev);
#pragma unroll
            for (int n = 0; n < NT; ++n)
            {
                // both positions of a row (integers), both rows of a position (halves), at a time
                const float2 u = make_float2(f[n][0] * uk, f[n][RT - 1] * uk), both = make_float2(add, add);
                const float2 u_high = mul2(u, make_float2(p.scale, p.scale)), u_low = mul2(u, make_float2(p.scale_low, p.scale_low));
                if constexpr (kInt) {
                    const float2 x = make_float2(c4[n][0], c4[n][2]), z = fma2(x, u_high, fma2(x, u_low, both));
                    s[b][n][0][0] = z.x;
                    s[b][n][1][0] = z.y;
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = make_float2(c4[n][2 * h], c4[n][2 * h + 1]), z = fma2(x, u_high, fma2(x, u_low, both));
                        s[b][n][h][0] = z.x;
                        s[b][n][h][RT - 1] = z.y;
                    }
                }
            }
            const int page = at + b;
            if (id[b] < 0 || page < whole_first || page >= whole_last) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < RT; ++k) {
                        const int low = p.window ? pos[n][k] - p.window : -1;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int key = page * kKv8Block + g + 8 * h;
                            if (id[b] < 0 || key > pos[n][k] || key <= low) s[b][n][h][k] = -INFINITY;
                        }
                    }
            }
        }
        bool moved = false;
        float c[NT][RT], top[NT][RT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < RT; ++k) {
                float x = m[n][k];
#pragma unroll
                for (int b = 0; b < PB; ++b) x = fmaxf(x, fmaxf(s[b][n][0][k], s[b][n][1][k]));
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(kFull, x, w));
                c[n][k] = m[n][k] == x ? 1.0f : ex2(m[n][k] - x);
                moved |= m[n][k] != x;
                m[n][k] = x;
                top[n][k] = x == -INFINITY ? 0.0f : kInt ? x : x - kKv8WeightBits;  // nothing seen yet: weights 2^(-inf - 0)
                l[n][k] *= c[n][k];
            }
        if constexpr (kInt) {
            uint32_t high[PB], low[PB];  // B fragments: the weights' bytes of column g, four positions a page
#pragma unroll
            for (int b = 0; b < PB; ++b) {
                uint32_t w[2];
                float sum = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float weight = ex2(s[b][0][h][0] - top[0][0]);
                    sum += weight;
                    w[h] = __float2uint_rn(weight * kKv8FixedScale);
                }
                l[0][0] = fmaf(sum, less[b], l[0][0]);
                // bytes 2, 3 and 0, 1 of positions g and g + 8 to the lanes that multiply them
                const uint32_t upper = __byte_perm(w[0], w[1], 0x7632), lower = __byte_perm(w[0], w[1], 0x5410);
                high[b] = __byte_perm(__shfl_sync(kFull, upper, from0), __shfl_sync(kFull, upper, from1), pick);
                low[b] = __byte_perm(__shfl_sync(kFull, lower, from0), __shfl_sync(kFull, lower, from1), pick);
            }
            int base[4] = {0, 0, 0, 0}, base_low[4] = {0, 0, 0, 0};  // of the output's sums
#pragma unroll
            for (int b = 0; b < PB; b += 2) {
                imma_s8_u8(base, base, kKv8Minus128, kKv8Minus128, kKv8Minus128, kKv8Minus128, high[b], high[b + 1]);
                imma_s8_u8(base_low, base_low, kKv8Minus128, kKv8Minus128, kKv8Minus128, kKv8Minus128, low[b], low[b + 1]);
            }
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                uint4 v[PB];
#pragma unroll
                for (int b = 0; b < PB; ++b)
                    v[b] = *reinterpret_cast<const uint4*>(pages_at + b * kPageBytes + kKv8Block * D + j * 512 + lane * 16);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    int x[4], y[4];
#pragma unroll
                    for (int b = 0; b < PB; b += 2) {
                        const uint32_t a0 = k ? v[b].z : v[b].x, a1 = k ? v[b].w : v[b].y;
                        const uint32_t a2 = k ? v[b + 1].z : v[b + 1].x, a3 = k ? v[b + 1].w : v[b + 1].y;
                        imma_u8_u8(x, b ? x : base, a0, a1, a2, a3, high[b], high[b + 1]);
                        imma_u8_u8(y, b ? y : base_low, a0, a1, a2, a3, low[b], low[b + 1]);
                    }
                    const float2 upper = make_float2(static_cast<float>(x[0] * 256 + x[1]), static_cast<float>(x[2] * 256 + x[3]));
                    const float2 lower = make_float2(static_cast<float>(y[0] * 256 + y[1]), static_cast<float>(y[2] * 256 + y[3]));
                    const float2 z = fma2(make_float2(o[2 * j + k][0][0], o[2 * j + k][0][1]), make_float2(c[0][0], c[0][0]),
                                          fma2(upper, make_float2(65536.0f, 65536.0f), lower));
                    o[2 * j + k][0][0] = z.x;
                    o[2 * j + k][0][1] = z.y;
                }
            }
        } else {
            uint32_t ph[PB][NT][2], pl[PB][kFine ? NT : 1][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < PB; ++b) {
                    float w[2][RT];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 z = add2(make_float2(s[b][n][h][0], s[b][n][h][RT - 1]), make_float2(-top[n][0], -top[n][RT - 1]));
                        w[h][0] = ex2(z.x);
                        w[h][RT - 1] = ex2(z.y);
                    }
                    const float2 sum = fma2(add2(make_float2(w[0][0], w[0][RT - 1]), make_float2(w[1][0], w[1][RT - 1])),
                                            make_float2(less[b], less[b]), make_float2(l[n][0], l[n][RT - 1]));
                    l[n][0] = sum.x;
                    l[n][RT - 1] = sum.y;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t high = half2_bits(w[h][0], w[h][RT - 1]);
                        ph[b][n][h] = movmatrix_trans(high);
                        if constexpr (kFine) {
                            const float2 r = half2_floats(high ^ 0x80008000u);
                            const float2 rest = add2(make_float2(w[h][0], w[h][RT - 1]), r);
                            pl[b][n][h] = movmatrix_trans(half2_bits(rest.x, rest.y));
                        }
                    }
                }
            if (__any_sync(kFull, moved)) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < OT; j += 2) {
                            const float2 z = mul2(make_float2(o[k][n][j], o[k][n][j + 1]), make_float2(c[n][0], c[n][RT - 1]));
                            o[k][n][j] = z.x;
                            o[k][n][j + 1] = z.y;
                        }
            }
            if constexpr (!kInt) {
#pragma unroll
                for (int b = 0; b < PB; ++b)
#pragma unroll
                    for (int j = 0; j < D / 32; ++j) {
                        const uint4 w4 = *reinterpret_cast<const uint4*>(pages_at + b * kPageBytes + kKv8Block * D + j * 512 + lane * 16);
                        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t a0 = kv8_halves<false>(w[2 * k]), a1 = kv8_halves<false>(w[2 * k + 1]);
                            const uint32_t a2 = kv8_halves<true>(w[2 * k]), a3 = kv8_halves<true>(w[2 * k + 1]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma16816(o[2 * j + k][n], a0, a1, a2, a3, ph[b][n][0], ph[b][n][1]);
                                if constexpr (kFine) mma16816(o[2 * j + k][n], a0, a1, a2, a3, pl[b][n][0], pl[b][n][1]);
                            }
                        }
                    }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring becomes the warps' results

    // the warps' shares meet
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < RT; ++k) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[n][k] += __shfl_xor_sync(kFull, l[n][k], w);
            const int r = kInt ? t : n * 8 + 2 * t + k;
            if (g == 0) s_ml[warp][r] = make_float4(m[n][k], l[n][k], __int_as_float(ref), 0.0f);
            if (r >= n_rows) continue;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const float* x = o[2 * j][n];
                const float* y = o[2 * j + 1][n];
                *reinterpret_cast<float4*>(&s_o[warp][r][32 * j + 4 * g]) =
                    kInt ? make_float4(x[0], x[1], y[0], y[1]) : make_float4(x[k], x[OT - 2 + k], y[k], y[OT - 2 + k]);
            }
        }
    // The hidden pages in fp32, into the warp's share: the windows once more.
    __syncwarp();
    if (s_range[warp].w) {
        const int unit_ref = ref;
        int4 range = start();
        for (int window = 0; first + warp * PB + window * kStep < last; window += kTurns) {
            fetch(0, window);
            const int away = look(range);
            for (unsigned left = __ballot_sync(kFull, away >= 0); left; left &= left - 1) {
                const int from = __ffs(left) - 1, ex = __shfl_sync(kFull, scales[0], from);
                const int page = first + warp * PB + (window + from / PB) * kStep + from % PB;
                const uint8_t* block = base + __shfl_sync(kFull, away, from) * page_bytes;
                const float uk = __int_as_float((ex & 0xff) << 23);
                const float unit = (kInt ? kKv8FixedScale : 1.0f) * pow2i((ex >> 8) - unit_ref);  // of a weight in O, and the value scale
#pragma unroll 1
                for (int r = 0; r < n_rows; ++r) {
                    const int of = token(rho0 + r), position = at0 + of, key = page * kKv8Block + (lane & 15);
                    const size_t row = static_cast<size_t>(sq.row0 + of) * p.q_stride +
                                       static_cast<size_t>(head * p.group.d + rho0 + r - of * p.group.d) * D;
                    // half the score of position lane % 16
                    float dot = 0.0f;
#pragma unroll 2
                    for (int d = (lane >> 4) * (D / 2); d < ((lane >> 4) + 1) * (D / 2); d += 4) {
                        const float4 x = load_row4<kBf16>(p.q, row + d);
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(block + (lane & 15) * D + d);
                        dot = fmaf(x.x, kv8_number(w, 0), fmaf(x.y, kv8_number(w, 1), fmaf(x.z, kv8_number(w, 2), fmaf(x.w, kv8_number(w, 3), dot))));
                    }
                    dot = (dot + __shfl_xor_sync(kFull, dot, 16)) * uk;
                    float z = fmaf(dot, p.scale, dot * p.scale_low);
                    if (key > position || (p.window && key <= position - p.window)) z = -INFINITY;
                    const float4 ml = s_ml[warp][r];
                    float now = z;
#pragma unroll
                    for (int w = 1; w < 16; w <<= 1) now = fmaxf(now, __shfl_xor_sync(kFull, now, w));
                    now = fmaxf(now, ml.x);
                    const float by = ml.x == now ? 1.0f : ex2(ml.x - now);
                    const float weight = ex2(z - (now == -INFINITY ? 0.0f : kInt ? now : now - kKv8WeightBits)), each = weight * unit;
                    float sum = weight;
#pragma unroll
                    for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(kFull, sum, w);
#pragma unroll 1
                    for (int j = 0; j < D / 32; ++j) {  // dim 32j + lane
                        float& to = s_o[warp][r][j * 32 + lane];
                        float x = to * by;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t v = *reinterpret_cast<const uint32_t*>(block + kKv8Block * D + j * 512 + g * 64 + w * 16 + t * 4);
#pragma unroll
                            for (int k = 0; k < 4; ++k) x = fmaf(__shfl_sync(kFull, each, kv8_value_pos(w, k)), kv8_number(v, k), x);
                        }
                        to = x;
                    }
                    __syncwarp();
                    if (lane == 0) s_ml[warp][r] = make_float4(now, ml.y * by + sum, ml.z, 0.0f);
                    __syncwarp();
                }
            }
        }
    }
    __syncthreads();
    constexpr int kQuads = D / 4;
    constexpr float kUnit = kInt ? 1.0f / kKv8FixedScale : 1.0f;
    for (int x = threadIdx.x; x < n_rows * kQuads; x += 32 * kWarps) {
        const int r = x / kQuads, d = x % kQuads * 4;
        Kv8Share s = kv8_nothing();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) kv8_fold(s, s_ml[w][r], *reinterpret_cast<const float4*>(&s_o[w][r][d]));
        if (active == 1) {
            const float inv = kv8_inverse(s.l, s.ref, kUnit);
            kv8_store<D, kBf16>(p, sq.row0, rho0 + r, head, d, make_float4(s.a.x * inv, s.a.y * inv, s.a.z * inv, s.a.w * inv));
        } else {
            const size_t at_part = (static_cast<size_t>(item) * p.splits + split) * kRows + r;
            *reinterpret_cast<float4*>(p.part + at_part * D + d) = s.a;
            if (d == 0) p.part_ml[at_part] = make_float4(s.m, s.l, __int_as_float(s.ref), 0.0f);
        }
    }
    if (active == 1) return;
    kv8_merge<D, kBf16, 32 * kWarps, 1>(p, kUnit, [] { __syncthreads(); }, reinterpret_cast<float4*>(s_ring), &s_last, item, active, kRows,
                                        n_rows, sq.row0, rho0, head);
}

}  // namespace phonon
