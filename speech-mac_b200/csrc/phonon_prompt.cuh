// Causal attention over packed prompts (sm_100a): the row at position p of a
// prompt sees its positions (p - window, p], all up to p without a window.
//
//   out[p] = sum_j softmax_j(scale q[p] . k[j]) v[j]
//
// Rows lie packed, prompt i in rows [row_begin[i], row_begin[i + 1]), and
// query heads are grouped on K/V heads.
#pragma once

#include "phonon_head_gemm.cuh"
#include "phonon_i8.cuh"

namespace phonon {

struct PromptParams {
    const void *q, *k, *v;  // [rows][heads][D], [rows][kv_heads][D] twice; rows `stride` elements apart
    void* out;
    long long q_stride, k_stride, v_stride, out_stride;
    const int32_t* begin;  // [prompts + 1]
    int32_t* status;       // [prompts] or null
    int prompts, rows, max_rows, heads, kv_heads;
    Kv8Div group;     // query heads of a K/V head
    int window;       // 0: none
    float scale;      // times log2(e)
    Kv8Div pack;      // query heads that share a tile's rows: all of a K/V head's, or one
    int tokens;       // positions of a CTA
    Kv8Div by_tokens;
    int half;         // positions of a row tile: a CTA has one or two
    Kv8Div by_heads;  // CTAs of a tile
};

__device__ __forceinline__ void prompt_flag(const PromptParams& p, int i, int code) {
    if (p.status) atomicMax(p.status + i, code);
}

// The slot-th tile of the call: the `tokens` positions of a prompt that a CTA
// works on, the last ones first (they see most). index < 0: the call has fewer.
struct PromptTile {
    int index, row0, length, first;  // prompt, its first row and rows, the tile's first position
};

// A prompt whose rows lie outside the call's, are more than max_rows or begin
// before an earlier prompt's has none: tiles never share rows, and there are at
// most rows / tokens + prompts of them, one less for every prompt without.
// `report`: one CTA of the last slot, which reads all prompts if there is such
// a one. One warp, 128 prompts at a time.
__device__ __forceinline__ void prompt_find(const PromptParams& p, int slot, bool report, PromptTile* out) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) out->index = -1;
    __syncwarp();
    int before = 0, most = 0;  // tiles and the largest begin of the prompts so far
    int x[5], next[5];
    const auto load = [&](int (&y)[5], int base) {
#pragma unroll
        for (int k = 0; k < 5; ++k) y[k] = base < p.prompts ? p.begin[min(base + 4 * lane + k, p.prompts)] : 0;
    };
    load(x, 0);
    for (int base = 0; base < p.prompts; base += 128) {
        load(next, base + 128);
        const int i = base + 4 * lane;
        int top = max(max(x[0], x[1]), max(x[2], x[3]));  // (of prompts behind the last: the last's end, which is no begin of theirs)
        int highest = top;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, highest, o);
            if (lane >= o) highest = max(highest, y);
        }
        int earlier = __shfl_up_sync(kFull, highest, 1);
        earlier = max(most, lane ? earlier : 0);
        int tiles[4], mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int b = x[k], e = x[k + 1];
            const bool good = b >= earlier && e >= b && e <= p.rows && e - b <= p.max_rows;
            if (i + k < p.prompts && !good && report) prompt_flag(p, i + k, kStatusInvalid);
            tiles[k] = i + k < p.prompts && good ? static_cast<int>(kv8_div(static_cast<uint32_t>(e - b + p.tokens - 1), p.by_tokens)) : 0;
            mine += tiles[k];
            earlier = max(earlier, b);
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, sum, o);
            if (lane >= o) sum += y;
        }
        int at = slot - (before + sum - mine);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at >= 0 && at < tiles[k]) *out = PromptTile{i + k, x[k], x[k + 1] - x[k], (tiles[k] - 1 - at) * p.tokens};
            at -= tiles[k];
        }
        before += __shfl_sync(kFull, sum, 31);
        most = max(most, __shfl_sync(kFull, highest, 31));
        if (slot < before) break;
#pragma unroll
        for (int k = 0; k < 5; ++k) x[k] = next[k];
    }
}

// Piece `piece` (16 bytes) of a staged row of kRow bytes: pieces are turned so
// that neither a row's nor a piece of all rows share banks.
template <int kRow>
__device__ __forceinline__ uint32_t prompt_staged(uint32_t staging, int row, int piece) {
    return staging + row * kRow + ((piece ^ (kRow == 64 ? row >> 1 & 3 : row & (kRow / 16 - 1))) * 16);
}

__device__ __forceinline__ float4 prompt_get16(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}

// A lane's staged row of kRow bytes, fp32 or bf16: infinities become the largest
// number of their sign. (Not unrolled: few rows come here.)
template <int kRow, bool kBf16>
__device__ __forceinline__ void prompt_within(uint32_t staging) {
#pragma unroll 1
    for (int k = 0; k < kRow; k += 4) {
        const uint32_t at = prompt_staged<kRow>(staging, threadIdx.x & 31, k / 16) + k % 16;
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at));
        w -= kBf16 ? __vcmpeq2(w & 0x7fff7fffu, 0x7f807f80u) & 0x00010001u : (w & 0x7fffffffu) == 0x7f800000u;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
    }
}

// A warp's 32 staged rows (of kRow bytes) to the output, whole sectors at a
// time. own: the byte of the output that the lane's row goes to, or -1.
template <int kRow>
__device__ __forceinline__ void prompt_put_rows(void* out, long long own, uint32_t staging) {
    constexpr int kPieces = kRow / 16, kEach = 32 / kPieces;
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < 32; i += kEach) {
        const int r = i + lane / kPieces;
        const long long at = __shfl_sync(kFull, own, r);
        const float4 x = prompt_get16(prompt_staged<kRow>(staging, r, lane % kPieces));
        if (at >= 0) *reinterpret_cast<float4*>(static_cast<uint8_t*>(out) + at + lane % kPieces * 16) = x;
    }
    __syncwarp();
}

// ------------------------------------------------- bf16 rows on tcgen05
// A CTA has two row tiles (one, where that leaves SMs without) of 128 rows (a row is a position and one of the
// `pack` query heads that share its K/V head), each with a softmax of four
// warps, a row a thread: while one tile's scores become weights, the tensor
// cores work for another.
//
//   warp 8     brings q, then 64 or 128 positions of k and of v a turn by TMA
//   warp 9     (and 10) issues S = q k^T and O += P v of the tiles
//   warps 0-7  S to registers, its maximum, the weights 2^(s - M) as bf16 back
//              over S (the A operand of P v), the sum of weights in fp32
//
// Weights are rounded to bf16, as the matrix instruction wants them beside bf16
// values. It shows: an output's error against 64 bits is 1.95e-3 (prompts of up
// to 512) to 2.2e-3 (of 8191, or a window of 250) of the outputs' norm, where
// rounding the output alone makes 1.62e-3 to 1.66e-3. Two slices a weight bring
// it down to that and take 13 % (64 dims, short) to 30 % (128 dims, long) more
// time; the sum of the rounded weights in place of the exact ones makes no
// difference that shows (1.97e-3 and 1.95e-3 in a model of 2000 positions) and
// takes 4 % more with 128 dims. Rows in fp32 lose nothing.
//
// O stays in TMEM. M follows the maximum only where that would make weights
// above 2^8: the tile's own warps then multiply O by 2^(M - M'), which they may
// since S of a turn comes behind P v of the turn before in the tensor cores'
// order.
//
// Positions that a row does not see get the weight 0, whose product with a v
// that is not finite is NaN. So where an output is not finite the CTA starts
// over, carefully: warp 8 looks at every turn's values, puts 0 in place of
// those that are not finite, and the rows that see one become NaN. And O, which
// is divided by the sum of weights at the end, may leave fp32's range where the
// mean of the values does not (weights up to 2^8 times any value, over all
// keys), so that pass has the values times a power of two: exact, but for
// values below 2^-60, some of whose bits may be lost beside the others.
// (Nothing is written before: out may lie over q. The pass has barriers of its
// own; none is ever set up twice. Both passes are a loop over the same code, and
// what the second adds is kept small: more of it, behind branches that are not
// taken, took calls with 128 dims 5 % longer.)
//
// Measured: prompts of 8191 and 7500, 32 heads on 8 x 128: 880 us where a
// captured graph has a few of them, 1.2 PFLOP/s of the products that rows see (73
// % of the measured matrix rate), 1030 in a long loop of calls, under the power
// limit (1.03; 74 % of the sustained rate). 4 of 4096 in a graph: 16 heads of 128
// 265 to 300 us, of 64 212 (1.0 and 0.65 PFLOP/s). With 128 dims
// matrix and exponential units are each busy half of the time, and the two
// tiles' turns do not fill each other's gaps; with 64 the exponentials are the
// most. 64 prompts of up to 512 take 40 us and 16 with a window of 250 61, bound
// by a turn's chain (S, its maximum, weights, P v: 2000 clocks and more) and
// a CTA's start and end (4000), four tiles an SM.
constexpr int kPromptThreads = 384;
constexpr float kPromptSlack = 8.0f;

// 128 dims: 128 positions a turn, TMEM and registers of an SM for one CTA. Up
// to 64 dims the exponentials are the most of the work, and 64 positions a turn
// leave room for two CTAs: four tiles' softmaxes to keep their unit at work.
template <int D>
struct PromptShape {
    static constexpr int kBox = D < 64 ? D : 64, kBoxBytes = 2 * kBox, kBoxes = D / kBox;  // a row's piece of a tile
    static constexpr int kCtas = D == 128 ? 1 : 2, kKeys = D == 128 ? 128 : 64, kIssuers = kCtas;
    static constexpr int kStages = D == 128 ? 2 : 4, kTmemCols = 512 / kCtas;
    static constexpr int kQTile = 128 * D * 2, kTile = kKeys * D * 2;  // bytes of a row tile of q, of a turn's keys or values
    static constexpr int kSmem = 1024 + 2 * kQTile + 2 * kStages * kTile;
    // A thread's registers in warps 0-7 and 8-11, together what the launch has for each.
    static constexpr int kSoftmaxRegisters = kCtas == 1 ? 208 : 96, kOtherRegisters = kCtas == 1 ? 88 : 48;
    static constexpr int kRegisters = 256 * kSoftmaxRegisters + 128 * kOtherRegisters;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Rows of kBytes (128 or 64) in the swizzle of that width, 8 rows together. K
// major: the operand's K runs along the rows. MN major: it runs across them,
// blocks of kBytes of the other dimension `block` bytes apart.
template <int kBytes>
__device__ __forceinline__ uint64_t umma_desc_rows(uint32_t addr, uint32_t block = 16) {
    uint64_t d = (static_cast<uint64_t>(addr) >> 4) & 0x3FFFull;
    d |= static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16;     // leading byte offset
    d |= static_cast<uint64_t>(8 * kBytes >> 4) << 32;            // stride byte offset
    d |= static_cast<uint64_t>(1) << 46;                          // descriptor version (sm_100)
    d |= static_cast<uint64_t>(kBytes == 128 ? 2 : 4) << 61;      // SWIZZLE_128B, SWIZZLE_64B
    return d;
}

// k of the 2^-k that keeps a sum over `keys` weights up to 2^over times any
// values below 2^126.
__device__ __forceinline__ int prompt_down(int keys, int over) { return 34 - __clz(keys) + over; }

__device__ __forceinline__ float prompt_pow2(int e) { return __int_as_float((127 + e) << 23); }

constexpr uint32_t kUmmaBMnMajor = 1u << 16;  // of an instruction descriptor

// 16 packed columns of the warp's 32 lanes into TMEM.
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Two bf16 times 2^-down.
__device__ __forceinline__ uint32_t bf16x2_smaller(uint32_t w, int down) {
    const uint32_t by = (127 - down) * 0x800080u;
    const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&by));
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t bf16x2_bits(float a, float b) {  // a in the low half
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Which of the 32 keys from `key` on the row at `position` sees: bits.
__device__ __forceinline__ uint32_t prompt_seen(int position, int window, int key) {
    const int ahead = position - key, behind = window ? ahead - window : -1;  // sees keys (behind, ahead]
    uint32_t bits = ahead >= 31 ? kFull : ahead < 0 ? 0u : (2u << ahead) - 1;
    if (behind >= 0) bits &= behind >= 31 ? 0u : ~((2u << behind) - 1);
    return bits;
}

// The keys that the positions [first, end) see, in turns of kKeys from key0 on: [begin, end).
struct PromptTurns {
    int begin, end;
};
template <int kKeys>
__device__ __forceinline__ PromptTurns prompt_turns(int first, int end, int window, int key0) {
    if (end <= first) return {0, 0};
    const int low = window ? max(0, first - window + 1) : 0;
    return {(low - key0) / kKeys, (end - key0 + kKeys - 1) / kKeys};
}

template <int D>
__global__ void __launch_bounds__(kPromptThreads, PromptShape<D>::kCtas)
    prompt_bf16_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, PromptParams p) {
    using Shape = PromptShape<D>;
    constexpr int kStages = Shape::kStages, kTile = Shape::kTile, kQTile = Shape::kQTile, kBoxes = Shape::kBoxes, kBytes = Shape::kBoxBytes;
    constexpr int kKeys = Shape::kKeys, kIssuers = Shape::kIssuers, kParts = kKeys / 64;  // the weights go off 64 positions at a time
    constexpr int kWide = Shape::kCtas == 1 ? 4 : 1;  // 8 columns of O that registers are free for
    constexpr uint32_t kTmemO = 2 * kKeys;  // S of both tiles, the weights over it, then O
    static_assert(kTmemO + 2 * D <= Shape::kTmemCols, "TMEM");
    extern __shared__ uint8_t smem_raw[];
    constexpr uint32_t kBars = 4 * kStages + 2 * kParts + 7;
    __shared__ __align__(8) uint64_t s_bars[2 * kBars];
    __shared__ uint32_t s_tmem;
    __shared__ PromptTile s_tile;
    __shared__ int s_failed, s_dirty;
    __shared__ uint32_t s_bad[kStages][kKeys / 32];  // careful: which of a turn's values are not finite
    const uint32_t s_q = (smem_addr(smem_raw) + 1023) & ~1023u, s_k = s_q + 2 * kQTile, s_v = s_k + kStages * kTile;
    uint32_t bars = smem_addr(s_bars);  // of this pass
    const auto k_full = [&] { return bars; };
    const auto k_empty = [&] { return bars + 8 * kStages; };
    const auto v_full = [&] { return bars + 16 * kStages; };
    const auto v_empty = [&] { return bars + 24 * kStages; };
    // by tile: S is there; the weights are (by part); the last P v is done
    const auto s_full = [&] { return bars + 32 * kStages; };
    const auto p_full = [&] { return bars + 32 * kStages + 16; };
    const auto o_full = [&] { return bars + 32 * kStages + 16 + 16 * kParts; };
    const auto q_full = [&] { return bars + 32 * kStages + 32 + 16 * kParts; };
    const auto tail = [&] { return q_full() + 8; };
    const auto idle = [&] { return q_full() + 16; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Two sets: one for each of the CTA's passes.
    if (threadIdx.x == 32) {
        for (uint32_t set = 0; set < 2; ++set) {
            const auto init = [&](uint32_t bar, int n, uint32_t count) {
                for (int x = 0; x < n; ++x) mbar_init(bar + 8 * (set * kBars + x), count);
            };
            init(k_full(), kStages, 1);
            init(k_empty(), kStages, kIssuers);
            init(v_full(), kStages, 1);
            init(v_empty(), kStages, kIssuers);
            init(s_full(), 2, 1);
            init(p_full(), 2 * kParts, 4);
            init(o_full(), 4, 1);  // and q_full(), tail()
            init(idle(), 1, kIssuers);
        }
        s_failed = s_dirty = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int slot = static_cast<int>(kv8_div(blockIdx.x, p.by_heads)), part = static_cast<int>(blockIdx.x - slot * p.by_heads.d);
    if (warp == 0) prompt_find(p, slot, blockIdx.x == gridDim.x - 1, &s_tile);
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(Shape::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_trigger();  // (not before: the next launch's CTAs, which wait for this one's end, may take TMEM where there is any left)
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const PromptTile t = s_tile;
    const uint32_t tmem = s_tmem;
    const auto free_tmem = [&] {
        if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Shape::kTmemCols) : "memory");
    };
    if (t.index < 0) {
        free_tmem();
        return;
    }
    const int pack = static_cast<int>(p.pack.d), head0 = part * pack, kv_head = static_cast<int>(kv8_div(head0, p.group));
    const int half = p.half, end = min(t.length, t.first + p.tokens);  // tile s: [first + s * half, min(end, first + (s + 1) * half))
    const int key0 = p.window ? max(0, t.first - p.window + 1) : 0;
    const PromptTurns turns0 = prompt_turns<kKeys>(t.first, min(end, t.first + half), p.window, key0);
    const PromptTurns turns1 = prompt_turns<kKeys>(t.first + half, end, p.window, key0);
    const int turns = max(turns0.end, turns1.end);
    const auto wait = [&](uint32_t bar, int use) {
        return __all_sync(kFull, mbar_wait(bar, use & 1, nullptr, &s_failed));
    };
    bool careful = false;
    const auto sync = [] {
        __syncwarp();
        asm volatile("bar.sync 1, %0;" ::"n"(kPromptThreads) : "memory");
    };
    // Every warp, at its end: whether the CTA starts over.
    const auto again = [&] {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        sync();
        if (careful || !s_dirty || s_failed) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bars += 8 * kBars;
        return careful = true;
    };
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kOtherRegisters));
        const bool two = turns1.end > 0;
        if (warp == 8) do {
            const auto load = [&](uint32_t to, const CUtensorMap* map, int rows, int head, int row, uint32_t bar) {
#pragma unroll
                for (int b = 0; b < kBoxes; ++b) tma_load_3d(to + b * rows * kBytes, map, b * Shape::kBox, head, row, bar);
            };
            if (lane == 0) {
                mbar_expect_tx(q_full(), (two ? 2 : 1) * half * pack * D * 2);
                load(s_q, &tm_q, 128, head0, t.row0 + t.first, q_full());
                if (two) load(s_q + kQTile, &tm_q, 128, head0, t.row0 + t.first + half, q_full());
            }
            int j = 0, looks = 0;
            for (; j < turns; ++j) {
                const int s = j % kStages, row = t.row0 + key0 + j * kKeys, there = end - key0 - j * kKeys;
                if (j >= kStages && !wait(k_empty() + 8 * s, j / kStages - 1)) break;
                if (lane == 0) {
                    mbar_expect_tx(k_full() + 8 * s, kTile);
                    load(s_k + s * kTile, &tm_k, kKeys, kv_head, row, k_full() + 8 * s);
                }
                if (j >= kStages && !wait(v_empty() + 8 * s, j / kStages - 1)) break;
                const bool look = careful || there < kKeys;  // what follows the prompt may not be finite: zeros
                const uint32_t bar = look ? tail() : v_full() + 8 * s;
                if (lane == 0) {
                    mbar_expect_tx(bar, kTile);
                    load(s_v + s * kTile, &tm_v, kKeys, kv_head, row, bar);
                }
                if (!look) continue;
                if (lane < kKeys / 32) s_bad[s][lane] = 0;
                if (!wait(tail(), looks++)) break;
                for (int x = lane; x < kKeys * kBoxes; x += 32) {  // a key's box each
                    const int key = x % kKeys;
                    const uint32_t at = s_v + s * kTile + x * kBytes;
                    bool bad = false;
                    for (int c = 0; c < kBytes; c += 16) {
                        uint32_t w[4] = {0, 0, 0, 0};
                        bool put = key >= there;
                        if (careful && !put) {
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + c));
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u, put = bad = true;
                                if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu, put = bad = true;
                            }
                        }
                        if (put) kv8_put16(at + c, w[0], w[1], w[2], w[3]);
                    }
                    if (bad) atomicOr(&s_bad[s][key >> 5], 1u << (key & 31));
                }
                if (careful) {
                    __syncwarp();
                    for (int x = lane; x < kTile / 4; x += 32) {
                        uint32_t w;
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(s_v + s * kTile + 4 * x));
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(s_v + s * kTile + 4 * x), "r"(bf16x2_smaller(w, prompt_down(end - key0, 8))) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full() + 8 * s);
            }
            if (j < turns && lane == 0) {  // a wait ran out: no copy is on its way when the CTA gives its memory back
                mbar_settle(q_full(), 0);
                mbar_settle_ring(k_full(), kStages, j + 1);
                mbar_settle_ring(v_full(), kStages, j + 1);
            }
            __syncwarp();
        } while (again());
        else if (warp < 9 + kIssuers) do {
            constexpr uint32_t idesc_s = umma_idesc_bf16(128, kKeys), idesc_o = umma_idesc_bf16(128, D) | kUmmaBMnMajor;
            constexpr int kSteps = kBytes / 32;  // of 16 dims in a row of a box
            const int own = __shfl_sync(kFull, warp - 9, 0);
            uint32_t leader;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(leader));
            const auto commit = [&](uint32_t bar) {
                if (leader) umma_commit(bar);
            };
            const uint64_t q_desc = umma_desc_rows<kBytes>(s_q), k_desc = umma_desc_rows<kBytes>(s_k);
            const uint64_t v_desc = umma_desc_rows<kBytes>(s_v, kKeys * kBytes);
            bool ok = wait(q_full(), 0);
            int keys = 0, values = 0;  // turns known to be there (a wait takes a hundred clocks even if it ends at once)
            const auto score = [&](int tile, int j, bool last) {
                const int s = j % kStages;
                if (!ok || (j >= keys && !(ok = wait(k_full() + 8 * s, j / kStages)))) return;
                keys = j + 1;
                const PromptTurns in = tile ? turns1 : turns0;
                if (j >= in.begin && j < in.end) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t q = q_desc + tile * (kQTile / 16), kk = k_desc + s * (kTile / 16);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_half<false>(leader, tmem + tile * kKeys, q + (k / kSteps * 128 * kBytes + k % kSteps * 32) / 16,
                                         kk + (k / kSteps * kKeys * kBytes + k % kSteps * 32) / 16, idesc_s, k != 0);
                    commit(s_full() + 8 * tile);
                }
                if (last) commit(k_empty() + 8 * s);
            };
            const auto sum = [&](int tile, int j, bool last) {
                const int s = j % kStages;
                if (!ok || (j >= values && !(ok = wait(v_full() + 8 * s, j / kStages)))) return;
                values = j + 1;
                // (and the keys that come next)
                if (j + 1 < turns && j + 1 >= keys && !(ok = wait(k_full() + 8 * ((j + 1) % kStages), (j + 1) / kStages))) return;
                if (j + 1 < turns) keys = j + 2;
                const PromptTurns in = tile ? turns1 : turns0;
                if (j >= in.begin && j < in.end) {
                    const uint64_t v = v_desc + s * (kTile / 16);
#pragma unroll
                    for (int h = 0; h < kParts; ++h) {
                        if (!(ok = wait(p_full() + 8 * (tile * kParts + h), j - in.begin))) return;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                        for (int k = 4 * h; k < 4 * h + 4; ++k)
                            umma_half<true>(leader, tmem + kTmemO + tile * D, tmem + tile * kKeys + k * 8, v + k * kBytes, idesc_o, j != in.begin || k != 0);
                    }
                    if (j + 1 == in.end) commit(o_full() + 8 * tile);
                }
                if (last) commit(v_empty() + 8 * s);
            };
            if constexpr (kIssuers == 2) {
                score(own, 0, true);
                for (int j = 0; ok && j < turns; ++j) {
                    sum(own, j, true);
                    if (j + 1 < turns) score(own, j + 1, true);
                }
            } else {
                score(0, 0, false);
                score(1, 0, true);
                for (int j = 0; ok && j < turns; ++j) {
                    const bool more = j + 1 < turns;
                    sum(0, j, false);
                    if (more) score(0, j + 1, false);
                    sum(1, j, true);
                    if (more) score(1, j + 1, true);
                }
            }
            commit(idle());  // no product is on its way when the CTA gives its memory back
            mbar_settle(idle(), 0);
            if (ok) {
                mbar_settle_ring(k_empty(), kStages, turns);
                mbar_settle_ring(v_empty(), kStages, turns);
            }
            __syncwarp();
        } while (again());
        else do {
        } while (again());
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kSoftmaxRegisters));
        const int tile = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const PromptTurns in = tile ? turns1 : turns0;
        const int first = t.first + tile * half, at = static_cast<int>(kv8_div(r, p.pack)), position = first + at;
        const int last = min(end, first + half) - 1;  // the tile's last position
        const uint32_t at_s = tmem + tile * kKeys + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t at_o = tmem + kTmemO + tile * D + (static_cast<uint32_t>(quarter * 32) << 16);
        const bool mine = at < half && position <= last;
        uint32_t w[D / 2];  // the row's output
        bool good = true;
        do {
            float m = -INFINITY, l = 0.0f;
            for (int j = in.begin; j < in.end; ++j) {
                wait(s_full() + 8 * tile, j - in.begin);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float s[kKeys / 32][32];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) tmem_start(at_s + 32 * c, s[c]);
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) tmem_arrived(s[c]);
                const int key = key0 + j * kKeys;
                if (key + kKeys - 1 > first || (p.window && key <= last - p.window)) {  // not all of it by every row
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        const uint32_t bits = prompt_seen(position, p.window, key + 32 * c);
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[c][k] = bits >> k & 1 ? s[c][k] : -INFINITY;
                    }
                }
                float top[kKeys / 32];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) {
                    top[c] = fmaxf(s[c][0], s[c][1]);
#pragma unroll
                    for (int k = 2; k < 32; k += 2) top[c] = max3(top[c], s[c][k], s[c][k + 1]);
                }
                const float now = (kParts == 2 ? fmaxf(max3(top[0], top[1], top[kParts]), top[2 * kParts - 1]) : fmaxf(top[0], top[1])) * p.scale;
                const bool move = now > m + kPromptSlack;
                if (__any_sync(kFull, move)) {
                    const float to = move ? now : m;
                    const float by = m == to ? 1.0f : ex2(m - to);
                    m = to;
                    l *= by;
                    if (j != in.begin) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 8 * kWide) {
                            uint32_t o[8 * kWide];
#pragma unroll
                            for (int k = 0; k < 8 * kWide; k += 8) tmem_ld8(at_o + c + k, o, k);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8 * kWide; k += 8) {
                                uint32_t x[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(__uint_as_float(o[k + i]) * by);
                                tmem_store8(at_o + c + k, x);
                            }
                        }
                    }
                }
                const float from = m == -INFINITY ? 0.0f : -m;  // nothing seen yet: weights 2^-inf
                const float2 scale = make_float2(p.scale, p.scale), from2 = make_float2(from, from);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < kParts; ++h) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t x[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float2 z = fma2(make_float2(s[2 * h + c][2 * k], s[2 * h + c][2 * k + 1]), scale, from2);
                            const float2 e = make_float2(ex2(z.x), ex2(z.y));
                            sum[k & 1] = add2(sum[k & 1], e);
                            x[k] = bf16x2_bits(e.x, e.y);
                        }
                        tmem_store16(at_s + 32 * h + 16 * c, x);
                    }
                    if (careful && h + 1 == kParts) {
                        wait(v_full() + 8 * (j % kStages), j / kStages);
                        for (int c = 0; c < kKeys / 32; ++c)
                            if (s_bad[j % kStages][c] & prompt_seen(position, p.window, key + 32 * c)) l = __int_as_float(0x7fc00000);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full() + 8 * (tile * kParts + h));
                }
                const float2 both = add2(sum[0], sum[1]);
                l += both.x + both.y;
            }
            if (in.end > in.begin) wait(o_full() + 8 * tile, 0);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float inverse = *static_cast<volatile int*>(&s_failed) ? __int_as_float(0x7fc00000) : __fdiv_rn(1.0f, l);
            if (careful) inverse *= prompt_pow2(prompt_down(end - key0, 8));
            const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
            __nv_bfloat162 clean = zero;  // NaN once an output is not finite
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float o[32];
                tmem_start(at_o + c, o);
                tmem_arrived(o);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    w[c / 2 + k] = bf16x2_bits(o[2 * k] * inverse, o[2 * k + 1] * inverse);
                    clean = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w[c / 2 + k]), zero, clean);
                }
            }
            good = !mine || __low2float(clean) + __high2float(clean) == 0.0f || (careful && inverse < INFINITY);
            if (!good) s_dirty = 1;
            __syncwarp();
        } while (again());
        // through q's room, which nothing reads any more
        const uint32_t staging = s_q + tile * kQTile + quarter * (32 * 2 * D);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) kv8_put16(prompt_staged<2 * D>(staging, lane, k), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        if (careful) prompt_within<2 * D, true>(staging);  // (means of finite values, that roundings have carried over the end)
        prompt_put_rows<2 * D>(p.out, mine ? 2 * ((t.row0 + position) * p.out_stride + (head0 + r - at * pack) * D) : -1, staging);
        if (!good) prompt_flag(p, t.index, s_failed ? kStatusDevice : kStatusNonFinite);
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    free_tmem();
}

// ------------------------------------------------- fp32 rows on tcgen05
// Every operand as three bf16 slices (8 bits each, the differences exact), and
// a product as the six slice products that are above 2^-24 of it, the smallest
// first: 6 times the matrix work, and fp32's precision. A CTA has one row tile
// of 128 rows and 64 positions a turn:
//
//   warps 8-15  read k and v, and write their slices as matrix operands
//   warps 4, 5  issue S = q k^T one or two turns ahead, and P v (one warp for both was
//               the slowest part: a wait takes it 200 clocks)
//   warps 0-3   a row a thread: q times the softmax scale into TMEM (the A
//               operand of S), S to weights, their slices back over S, and the
//               sum of P v over the turns in registers (the tensor cores' own
//               sum truncates: 24 truncations a turn stay near fp32's rounding,
//               thousands would not)
//
// Values that are not finite, sums that leave fp32's range: as for bf16 rows; of keys that are not, or would
// not be as bf16, the careful CTA computes the scores one by one.
//
// Measured, in a graph: 2 prompts of 4096, 16 heads of 128, 710 to 820 us by the
// power limit, 168 to 194 TFLOP/s of the products that rows see, 1.0 to 1.16
// PFLOP/s of slices (71 % of the measured matrix rate); of 64 400 us; 4 of 1024
// to 2048, 8 x 64, 90 us (97 among a user's calls). Long prompts are bound
// by the tensor cores; short ones by a CTA's start, end and chain of turns
// (one of 128: 9 us). Errors stay at or below those of the plain form in fp32
// (0.1 to 0.5e-6 of the output's norm against 0.1 to 1.2e-6).
constexpr int kPromptF32Threads = 512, kPromptF32Keys = 64;
// A thread's registers in warps 0-3 and 4-15, together the launch's 128 each.
constexpr int kPromptF32SoftmaxRegisters = 240, kPromptF32OtherRegisters = 88;
constexpr int kPromptF32Registers = 128 * kPromptF32SoftmaxRegisters + 384 * kPromptF32OtherRegisters;

template <int D>
struct PromptF32Shape {
    static constexpr int kBox = D < 64 ? D : 64, kBoxBytes = 2 * kBox, kBoxes = D / kBox;
    static constexpr int kStages = D == 128 ? 2 : 3;
    static constexpr int kBuffers = D == 128 ? 2 : 3;  // of S and the weights over it
    static constexpr int kPlane = kPromptF32Keys * D * 2;  // bytes of a slice of a turn's keys or values
    static constexpr int kChunk = D < 64 ? D : 64, kStaging = 128 * kChunk * 4;  // dims of 128 rows at a time, on their way in and out
    static constexpr int kSmem = 1024 + 2 * kStages * 3 * kPlane + kStaging;
    static constexpr int kUnits = D / 32;  // of 8 elements a converting thread has, of a turn's keys and of its values
    static constexpr int kBatch = kUnits < 2 ? kUnits : 2, kParts = kUnits / kBatch;  // of them at a time
};

// The three slices of a pair, the first in the low half; exact but for the
// last one's rounding.
__device__ __forceinline__ void bf16x2_slices(float2 x, uint32_t (&w)[3]) {
    w[0] = bf16x2_bits(x.x, x.y);
    const float2 minus = make_float2(-1.0f, -1.0f);
    x = fma2(make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u)), minus, x);
    w[1] = bf16x2_bits(x.x, x.y);
    x = fma2(make_float2(__uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)), minus, x);
    w[2] = bf16x2_bits(x.x, x.y);
}

// Slices of a product, smallest first.
__device__ __forceinline__ constexpr int prompt_slice_a(int i) { return i == 0 ? 2 : i == 1 || i == 3 ? 1 : 0; }
__device__ __forceinline__ constexpr int prompt_slice_b(int i) { return i == 2 ? 2 : i == 1 || i == 4 ? 1 : 0; }

constexpr float kBf16Most = 3.38953139e38f;  // the largest bf16

template <int D>
__global__ void __launch_bounds__(kPromptF32Threads, 1) prompt_f32_kernel(PromptParams p) {
    using Shape = PromptF32Shape<D>;
    constexpr int kStages = Shape::kStages, kPlane = Shape::kPlane, kBytes = Shape::kBoxBytes, kKeys = kPromptF32Keys, kBatch = Shape::kBatch, kParts = Shape::kParts, kBuffers = Shape::kBuffers;
    constexpr uint32_t kTmemS = 3 * D / 2, kSCols = 96, kTmemO = kTmemS + kBuffers * kSCols;  // q's slices, S with the weights' slices over it, O
    static_assert(kTmemO + D <= 512, "TMEM");
    extern __shared__ uint8_t smem_raw[];
    constexpr uint32_t kBars = 4 * kStages + kBuffers + 7;
    __shared__ __align__(8) uint64_t s_bars[2 * kBars];
    __shared__ uint32_t s_tmem;
    __shared__ PromptTile s_tile;
    __shared__ int s_failed, s_dirty;
    __shared__ unsigned long long s_bad[2][kStages];  // careful: which of a turn's keys, values are not finite
    const uint32_t s_k = (smem_addr(smem_raw) + 1023) & ~1023u, s_v = s_k + kStages * 3 * kPlane;
    uint32_t bars = smem_addr(s_bars);  // of this pass
    const auto k_full = [&] { return bars; };
    const auto k_empty = [&] { return bars + 8 * kStages; };
    const auto v_full = [&] { return bars + 16 * kStages; };
    const auto v_empty = [&] { return bars + 24 * kStages; };
    const auto s_full = [&] { return bars + 32 * kStages; };  // by buffer
    const auto p_full = [&] { return s_full() + 8 * kBuffers; };
    const auto o_full = [&] { return p_full() + 8; };  // P v of a turn: by turn % 4
    const auto q_full = [&] { return p_full() + 40; };
    const auto idle = [&] { return p_full() + 48; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Two sets: one for each of the CTA's passes.
    if (threadIdx.x == 32) {
        for (uint32_t set = 0; set < 2; ++set) {
            const auto init = [&](uint32_t bar, int n, uint32_t count) {
                for (int x = 0; x < n; ++x) mbar_init(bar + 8 * (set * kBars + x), count);
            };
            init(k_full(), kStages, 8);
            init(k_empty(), kStages, 1);
            init(v_full(), kStages, 8);
            init(v_empty(), kStages, 1);
            init(s_full(), kBuffers, 1);
            init(p_full(), 1, 4);
            init(o_full(), 4, 1);
            init(q_full(), 1, 4);
            init(idle(), 1, 2);
        }
        s_failed = s_dirty = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    const int slot = static_cast<int>(kv8_div(blockIdx.x, p.by_heads)), part = static_cast<int>(blockIdx.x - slot * p.by_heads.d);
    if (warp == 0) prompt_find(p, slot, blockIdx.x == gridDim.x - 1, &s_tile);
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_trigger();  // (not before: the next launch's CTAs, which wait for this one's end, may take TMEM where there is any left)
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const PromptTile t = s_tile;
    const uint32_t tmem = s_tmem;
    const auto free_tmem = [&] {
        if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    };
    if (t.index < 0) {
        free_tmem();
        return;
    }
    const int pack = static_cast<int>(p.pack.d), head0 = part * pack, kv_head = static_cast<int>(kv8_div(head0, p.group));
    const int end = min(t.length, t.first + p.tokens), key0 = p.window ? max(0, t.first - p.window + 1) : 0;
    const int turns = (end - key0 + kKeys - 1) / kKeys;
    const auto wait = [&](uint32_t bar, int use) {
        const bool ok = mbar_wait(bar, use & 1, nullptr, &s_failed);
        __syncwarp();
        return __all_sync(kFull, ok);
    };
    bool careful = false;
    const auto sync = [] {
        __syncwarp();
        asm volatile("bar.sync 1, %0;" ::"n"(kPromptF32Threads) : "memory");
    };
    // Every warp, at its end: whether the CTA starts over.
    const auto again = [&] {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        sync();
        if (careful || !s_dirty || s_failed) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bars += 8 * kBars;
        return careful = true;
    };
    if (warp >= 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptF32OtherRegisters));
        if (warp >= 8) do {
            // A warp writes whole rows' pieces: unit u of a turn's keys (values) is 8 dims of a row.
            constexpr int kChunks = D / 8;
            const int u0 = (warp - 8) * 32 + lane;
            const float* base[2] = {static_cast<const float*>(p.k) + static_cast<size_t>(t.row0 + key0) * p.k_stride + kv_head * D,
                                    static_cast<const float*>(p.v) + static_cast<size_t>(t.row0 + key0) * p.v_stride + kv_head * D};
            // batch n: the n-th of kParts pieces of a turn's keys, then of its values, then of the next turn
            const int batches = turns * 2 * kParts;
            const auto load = [&](float4 (&x)[kBatch][2], int n) {
                const int which = n / kParts & 1, j = n / (2 * kParts);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int u = u0 + 256 * (n % kParts * kBatch + i), row = j * kKeys + u / kChunks;
                    const float* at = base[which] + static_cast<size_t>(row) * (which ? p.v_stride : p.k_stride) + u % kChunks * 8;
                    const bool in = n < batches && key0 + row < end;  // what follows the prompt does not count: zeros
                    x[i][0] = in ? *reinterpret_cast<const float4*>(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[i][1] = in ? *reinterpret_cast<const float4*>(at + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            };
            bool ok = true;
            const auto put = [&](float4 (&x)[kBatch][2], int n) {
                const int which = n / kParts & 1, j = n / (2 * kParts), s = j % kStages;
                if (n >= batches) return;
                if (n % kParts == 0) {
                    if (j >= kStages) ok &= wait((which ? v_empty() : k_empty()) + 8 * s, j / kStages - 1);
                    if (careful) {  // (P v of the stage's last turn is behind what its rows read of s_bad)
                        if (j >= kStages) ok &= wait(v_empty() + 8 * s, j / kStages - 1);
                        if (u0 == 0) s_bad[which][s] = 0;
                        __syncwarp();
                        asm volatile("bar.sync 2, 256;" ::: "memory");
                    }
                }
                if (!ok) return;  // (every warp goes on to the last batch: they meet above)
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int u = u0 + 256 * (n % kParts * kBatch + i), row = u / kChunks, chunk = u % kChunks;
                    uint32_t w[4][3];
                    float* f = &x[i][0].x;
#pragma unroll
                    for (int k = 0; k < 4; ++k) bf16x2_slices(make_float2(f[2 * k], f[2 * k + 1]), w[k]);
                    if (careful) {
                        bool bad = false;
                        const float smaller = which ? prompt_pow2(-prompt_down(end - key0, 0)) : 1.0f;
#pragma unroll
                        for (int k = 0; k < 8; ++k) bad |= !(fabsf(f[k]) <= kBf16Most) && (!which || !isfinite(f[k]));
                        if (bad) atomicOr(&s_bad[which][s], 1ull << row);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            // numbers between the largest bf16 and the largest float keep their value
                            float2 y = make_float2(f[2 * k] * smaller, f[2 * k + 1] * smaller);
                            if (!isfinite(y.x)) y.x = 0.0f;
                            if (!isfinite(y.y)) y.y = 0.0f;
                            const float2 top = make_float2(fminf(fmaxf(y.x, -kBf16Most), kBf16Most), fminf(fmaxf(y.y, -kBf16Most), kBf16Most));
                            const bool far = top.x != y.x || top.y != y.y;
                            bf16x2_slices(far ? top : y, w[k]);
                            if (far) {
                                const float2 rest = make_float2(y.x - __uint_as_float(w[k][0] << 16), y.y - __uint_as_float(w[k][0] & 0xffff0000u));
                                w[k][1] = bf16x2_bits(rest.x, rest.y);
                                w[k][2] = bf16x2_bits(rest.x - __uint_as_float(w[k][1] << 16), rest.y - __uint_as_float(w[k][1] & 0xffff0000u));
                            }
                        }
                    }
                    const uint32_t at = (which ? s_v : s_k) + s * 3 * kPlane + chunk / (kBytes / 16) * kKeys * kBytes + row * kBytes +
                                        ((chunk % (kBytes / 16)) ^ (kBytes == 128 ? row & 7 : row >> 1 & 3)) * 16;
#pragma unroll
                    for (int c = 0; c < 3; ++c) kv8_put16(at + c * kPlane, w[0][c], w[1][c], w[2][c], w[3][c]);
                }
                if (n % kParts + 1 < kParts) return;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive((which ? v_full() : k_full()) + 8 * s);
            };
            float4 a[kBatch][2], b[kBatch][2], c[kBatch][2];
            load(a, 0);
            load(b, 1);
            load(c, 2);
            for (int n = 0; n < batches; n += 3) {
                put(a, n);
                load(a, n + 3);
                put(b, n + 1);
                load(b, n + 4);
                put(c, n + 2);
                load(c, n + 5);
            }
        } while (again());
        else if (warp <= 5) do {
            constexpr uint32_t idesc_s = umma_idesc_bf16(128, kKeys), idesc_o = umma_idesc_bf16(128, D) | kUmmaBMnMajor;
            uint32_t leader;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(leader));
            const auto commit = [&](uint32_t bar) {
                if (leader) umma_commit(bar);
            };
            const uint64_t k_desc = umma_desc_rows<kBytes>(s_k), v_desc = umma_desc_rows<kBytes>(s_v, kKeys * kBytes);
            constexpr int kSteps = kBytes / 32;  // of 16 dims in a row of a box
            bool ok = warp == 5 || wait(q_full(), 0);
            for (int j = 0; ok && j < turns; ++j) {
                const int s = j % kStages, before = j - kBuffers;
                const uint32_t at_s = tmem + kTmemS + j % kBuffers * kSCols;
                if (warp == 4) {
                    // (P v of that turn has read the weights that S goes over)
                    if (before >= 0) ok = wait(o_full() + 8 * (before & 3), before >> 2);
                    if (!ok || !(ok = wait(k_full() + 8 * s, j / kStages))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 6; ++i)
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
                            umma_half<true>(leader, at_s, tmem + prompt_slice_a(i) * (D / 2) + k * 8,
                                            k_desc + ((s * 3 + prompt_slice_b(i)) * kPlane + k / kSteps * kKeys * kBytes + k % kSteps * 32) / 16, idesc_s, (i | k) != 0);
                    commit(s_full() + 8 * (j % kBuffers));
                    commit(k_empty() + 8 * s);
                } else {
                    if (!(ok = wait(v_full() + 8 * s, j / kStages) && wait(p_full(), j))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 6; ++i)
#pragma unroll
                        for (int k = 0; k < kKeys / 16; ++k)
                            umma_half<true>(leader, tmem + kTmemO, at_s + prompt_slice_a(i) * (kKeys / 2) + k * 8,
                                            v_desc + ((s * 3 + prompt_slice_b(i)) * kPlane + k * 16 * kBytes) / 16, idesc_o, (i | k) != 0);
                    commit(o_full() + 8 * (j & 3));
                    commit(v_empty() + 8 * s);
                }
            }
            commit(idle());  // no product is on its way when the CTA gives its memory back
            mbar_settle(idle(), 0);
            if (ok) mbar_settle_ring(warp == 4 ? k_empty() : v_empty(), kStages, turns);
            __syncwarp();
        } while (again());
        else do {
        } while (again());
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptF32SoftmaxRegisters));
        const int r = threadIdx.x, at = static_cast<int>(kv8_div(r, p.pack)), position = t.first + at;
        const bool mine = at < p.tokens && position < end;
        const int head = head0 + r - at * pack;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        const float* q = static_cast<const float*>(p.q) + static_cast<size_t>(t.row0 + position) * p.q_stride + static_cast<size_t>(head) * D;
        const long long from_q = mine ? 4 * ((t.row0 + position) * p.q_stride + head * D) : -1;  // bytes
        const long long to_out = mine ? 4 * ((t.row0 + position) * p.out_stride + head * D) : -1;
        constexpr int kChunk = Shape::kChunk, kRow = 4 * kChunk, kPieces = kChunk / 4, kEach = 32 / kPieces;
        const uint32_t staging = s_v + kStages * 3 * kPlane + warp * (32 * kRow);
        float o[D];
        bool good = true;
        do {
            // q by whole sectors into shared memory, then its slices by rows. (Loops that are not unrolled here and
            // below: code that runs once a CTA is bound by its own instructions' way from memory.)
#pragma unroll 1
            for (int c = 0; c < D; c += kChunk) {
#pragma unroll 4
                for (int i = 0; i < 32; i += kEach) {
                    const int row = i + lane / kPieces;
                    const long long from = __shfl_sync(kFull, from_q, row);
                    copy16(prompt_staged<kRow>(staging, row, lane % kPieces),
                           static_cast<const uint8_t*>(p.q) + (from < 0 ? 0 : from + c * 4 + lane % kPieces * 16), from < 0 ? 0 : 16);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
#pragma unroll 1
                for (int k = 0; k < kPieces; k += 4) {
                    uint32_t w[3][8];
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float4 y = prompt_get16(prompt_staged<kRow>(staging, lane, k + i / 2));
                        uint32_t three[3];
                        bf16x2_slices(make_float2(y.x * p.scale, y.y * p.scale), three);
                        w[0][i] = three[0], w[1][i] = three[1], w[2][i] = three[2];
                        bf16x2_slices(make_float2(y.z * p.scale, y.w * p.scale), three);
                        w[0][i + 1] = three[0], w[1][i + 1] = three[1], w[2][i + 1] = three[2];
                    }
#pragma unroll
                    for (int i = 0; i < 3; ++i) tmem_store8(lanes + i * (D / 2) + c / 2 + 2 * k, w[i]);
                }
                __syncwarp();
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full());
#pragma unroll
            for (int k = 0; k < D; ++k) o[k] = 0.0f;
            float m = -INFINITY, l = 0.0f, shrink = 1.0f;
            const auto add_output = [&](int j) {
                wait(o_full() + 8 * (j & 3), j >> 2);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float2 by = make_float2(shrink, shrink);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    float x[32];
                    tmem_start(lanes + kTmemO + c, x);
                    tmem_arrived(x);
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float2 z = fma2(make_float2(o[c + k], o[c + k + 1]), by, make_float2(x[k], x[k + 1]));
                        o[c + k] = z.x;
                        o[c + k + 1] = z.y;
                    }
                }
            };
            for (int j = 0; j < turns; ++j) {
                const uint32_t at_s = lanes + kTmemS + j % kBuffers * kSCols;
                wait(s_full() + 8 * (j % kBuffers), j / kBuffers);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float s[2][32];
                tmem_start(at_s, s[0]);
                tmem_start(at_s + 32, s[1]);
                tmem_arrived(s[0]);
                tmem_arrived(s[1]);
                const int key = key0 + j * kKeys;
                if (careful) {
                    wait(k_full() + 8 * (j % kStages), j / kStages);
                    wait(v_full() + 8 * (j % kStages), j / kStages);
                    const unsigned long long seen = prompt_seen(position, p.window, key) |
                                                    static_cast<unsigned long long>(prompt_seen(position, p.window, key + 32)) << 32;
                    if (mine && s_bad[1][j % kStages] & seen) l = __int_as_float(0x7fc00000);
                    for (unsigned long long left = mine ? s_bad[0][j % kStages] & seen : 0; left; left &= left - 1) {
                        const int of = __ffsll(static_cast<long long>(left)) - 1;
                        const float* k_row = static_cast<const float*>(p.k) + static_cast<size_t>(t.row0 + key + of) * p.k_stride + kv_head * D;
                        float dot = 0.0f;
                        for (int d = 0; d < D; ++d) dot = fmaf(q[d] * p.scale, k_row[d], dot);
#pragma unroll
                        for (int k = 0; k < 64; ++k) s[k / 32][k % 32] = k == of ? dot : s[k / 32][k % 32];
                    }
                    __syncwarp();
                }
                if (key + kKeys - 1 > t.first || (p.window && key <= end - 1 - p.window)) {  // not all of it by every row
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t bits = prompt_seen(position, p.window, key + 32 * c);
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[c][k] = bits >> k & 1 ? s[c][k] : -INFINITY;
                    }
                }
                float top[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    top[c] = fmaxf(s[c][0], s[c][1]);
#pragma unroll
                    for (int k = 2; k < 32; k += 2) top[c] = max3(top[c], s[c][k], s[c][k + 1]);
                }
                const float now = max3(m, top[0], top[1]), c = m == now ? 1.0f : ex2(m - now);
                m = now;
                l *= c;
                const float from = now == -INFINITY ? 0.0f : -now;  // nothing seen yet: weights 2^-inf
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[3][16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float* x = &s[h][2 * k];
                        const float2 z = add2(make_float2(x[0], x[1]), make_float2(from, from));
                        const float2 e = make_float2(ex2(z.x), ex2(z.y));
                        sum = add2(sum, e);
                        uint32_t three[3];
                        bf16x2_slices(e, three);
                        w[0][k] = three[0], w[1][k] = three[1], w[2][k] = three[2];
                    }
#pragma unroll
                    for (int i = 0; i < 3; ++i) tmem_store16(at_s + i * (kKeys / 2) + h * 16, w[i]);
                }
                l += sum.x + sum.y;
                if (j) add_output(j - 1);
                shrink = c;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full());
            }
            add_output(turns - 1);
            float inverse = *static_cast<volatile int*>(&s_failed) ? __int_as_float(0x7fc00000) : __fdiv_rn(1.0f, l);
            if (careful) inverse *= prompt_pow2(prompt_down(end - key0, 0));
            float clean = 0.0f;  // NaN once an output is not finite
#pragma unroll
            for (int k = 0; k < D; ++k) {
                o[k] *= inverse;
                clean = fmaf(o[k], 0.0f, clean);
            }
            good = !mine || clean == 0.0f || (careful && inverse < INFINITY);
            if (!good) s_dirty = 1;
            __syncwarp();
        } while (again());
#pragma unroll
        for (int c = 0; c < D; c += kChunk) {
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
                kv8_put16(prompt_staged<kRow>(staging, lane, k), __float_as_uint(o[c + 4 * k]), __float_as_uint(o[c + 4 * k + 1]),
                          __float_as_uint(o[c + 4 * k + 2]), __float_as_uint(o[c + 4 * k + 3]));
            if (careful) prompt_within<kRow, false>(staging);
            prompt_put_rows<kRow>(p.out, to_out < 0 ? -1 : to_out + c * 4, staging);
        }
        if (!good) prompt_flag(p, t.index, s_failed ? kStatusDevice : kStatusNonFinite);
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    free_tmem();
}

}  // namespace phonon
