// Attention over the 8-bit cache for many rows (chunks of prompts) on the
// tcgen05 tensor cores.
//
// The mathematics is kv8_attention_kernel's: S = q K^T and O = P V with the
// held integers as halves, exact; the blocks' scales join S by columns of 16
// keys; the weights carry the blocks' value scales. A CTA has up to 256 rows
// of a K/V head and one split of its positions, 64 positions a turn:
//
//   warps 8-14  load the turns' bytes, a page's keys or values at a time, and
//               write them as halves into shared memory in matrix operand
//               order (8 rows of 16 bytes make a core matrix). The cache's
//               value order is kept: the 16 positions of a block come as
//               0 1 8 9 2 3 10 11 4 5 12 13 6 7 14 15 and the dims of 32 as
//               4g + w at column 8w + g. Sums over positions do not mind the
//               order as long as the weights have it too, and the dims are
//               put right when the output is stored.
//   warps 0-7   two streams of four warps, a row a thread, each with a
//               softmax, a score tile and an output tile of its own in TMEM:
//               the upper and the lower 128 rows of every turn, or, of up to
//               128 rows, every other turn each (their shares meet at the
//               end). S is read twice, for the maximum and for the weights,
//               which go back over S: the A operand of P V.
//   warp 15     issues S = q K^T and P V of whichever stream is ready, so that
//               one stream's products run under the other's softmax.
//
// P V of a turn is added to the O that the row's thread holds, in fp32
// registers and not in TMEM: a tensor core's sum truncates. 8 or 16
// truncations a turn stay below fp32's rounding of the whole, thousands of
// them one after another would not, and the maximum can move at any turn
// without a pass over TMEM.
//
// fp32 rows: q (times the softmax scale) and the weights as two halves each (22
// bits), two products each. bf16 rows: one half each (q's 8 bits are exact,
// weights keep 11). Blocks whose value scale is far from the split's smallest
// are hidden from the turns and added in fp32, a row a thread, at the end.
//
// 1024 rows a K/V head over 4096 positions, 32 heads: bf16, 128 dims 148 us
// (408 TFLOP/s of what rows see), fp32, 64 dims 134 us (225, twice that in
// products); the mma.sync kernel 353 and 265. Bound by the softmax's instructions: of 3000
// clocks a turn of 64 dims, 400 go to the maximum, 1300 to the weights (two
// warps share a scheduler's exponentials, 16 clocks an element of both), 250 to
// O, 250 to the wait for P V, 300 to barriers and loads; a start of 7500 clocks
// (4000 of them loads one after another: lengths, page ids, q and pages) and an
// end of 3000. Scores of 128 positions in one buffer a stream: 156 us in fp32,
// 134 in bf16. Warps that share a row's positions: 5300 clocks for 128.
#pragma once

#include "phonon_gemm.cuh"
#include "phonon_kv8.cuh"

namespace phonon {

constexpr int kKv8PromptKeys = 64, kKv8PromptStages = 4, kKv8PromptThreads = 512;
constexpr int kKv8Converters = 7;  // warps
// A thread's registers in warps 0-7 and 8-15, together the launch's 128 each.
constexpr int kKv8SoftmaxRegisters = 200, kKv8OtherRegisters = 56;
constexpr int kKv8PromptRegisters = 256 * (kKv8SoftmaxRegisters + kKv8OtherRegisters);
constexpr int kStatusDevice = 8;  // PHONON_CUDA_DEVICE_ERROR

// 32 consecutive accumulator columns of the warp's 32 lanes, on their way until tmem_arrived.
__device__ __forceinline__ void tmem_start(uint32_t taddr, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr)
        : "memory");
}

// All loads have arrived; r is not to be read before.
__device__ __forceinline__ void tmem_arrived(float (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
          "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
          "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
          "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
        :
        : "memory");
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {  // does not wait
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// Eight packed columns of the warp's 32 lanes into TMEM.
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// K-major operand without swizzle: core matrices of 8 rows x 16 bytes, the
// next along K 128 bytes on, the next 8 rows `rows8` bytes on.
__device__ __forceinline__ uint64_t umma_desc_plain(uint32_t addr, uint32_t rows8) {
    uint64_t d = (static_cast<uint64_t>(addr) >> 4) & 0x3FFFull;
    d |= static_cast<uint64_t>(128 >> 4) << 16;                          // leading byte offset
    d |= static_cast<uint64_t>((rows8 >> 4) & 0x3FFFu) << 32;            // stride byte offset
    d |= static_cast<uint64_t>(1) << 46;                                 // descriptor version (sm_100)
    return d;
}

// kind::f16 instruction descriptor: f32 accumulator, halves, both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_half(int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// A in shared memory (desc) or, kTmem, in TMEM (two halves a column). The whole
// warp runs this, so that operands stay in uniform registers; one lane issues.
template <bool kTmem>
__device__ __forceinline__ void umma_half(bool leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    if constexpr (kTmem)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
            "r"(static_cast<uint32_t>(a)), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(leader))
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(static_cast<uint32_t>(leader))
            : "memory");
}

__device__ __forceinline__ void kv8_put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void kv8_put8(uint32_t at, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Row tiles of 128 that a CTA has. Two share the turns' keys and values; q of
// fp32 rows of 128 dims takes two halves' room, where one tile fits.
template <int D, bool kBf16>
__host__ __device__ constexpr int kv8_prompt_tiles() { return D == 128 && !kBf16 ? 1 : 2; }

template <int D, bool kBf16>
__host__ __device__ constexpr int kv8_prompt_rows() { return 128 * kv8_prompt_tiles<D, kBf16>(); }

template <int D, bool kBf16>
__host__ __device__ constexpr int kv8_prompt_smem() {
    return (kBf16 ? 1 : 2) * kv8_prompt_rows<D, kBf16>() * D * 2 + 2 * kKv8PromptStages * kKv8PromptKeys * D * 2;
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kKv8PromptThreads, 1) kv8_prompt_kernel(Kv8AttnParams p) {
    constexpr int kTiles = kv8_prompt_tiles<D, kBf16>();
    constexpr int kKeys = kKv8PromptKeys, kPages = kKeys / kKv8Block, kStages = kKv8PromptStages;
    constexpr int kPlanes = kBf16 ? 1 : 2, kQBytes = 128 * D * 2, kTileBytes = kKeys * D * 2;
    constexpr uint32_t kRow8 = D * 16;      // bytes of 8 rows of q, of 8 keys
    constexpr uint32_t kDim8 = kKeys * 16;  // bytes of 8 dims of the values
    constexpr int kPieces = D / 32;         // 16-byte pieces a lane of a page's keys, of its values
    constexpr int kPitch = D + 4;           // floats of a row's result: 8 rows' quads in different banks
    static_assert(2 * 128 * kPitch * 4 <= kv8_prompt_smem<D, kBf16>(), "the rows' results outgrow the operands' room");
    extern __shared__ __align__(128) uint8_t s_mem[];  // q [tile][plane], kStages x keys, x values; then the rows' results
    __shared__ __align__(8) uint64_t s_bars[4 * kKv8PromptStages + 10];
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed, s_last, s_lo, s_hi;
    __shared__ float s_f[128 * kTiles];
    __shared__ float2 s_ml[2][128];  // M, sum
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t later = kv8_div(blockIdx.x, p.by_items), item = blockIdx.x - later * p.by_items.d;
    const uint32_t entry = kv8_div(item, p.by_heads);
    const int head = static_cast<int>(item - entry * p.by_heads.d);
    const int split = p.splits - 1 - static_cast<int>(later);
    const int i = static_cast<int>(kv8_div(entry, p.by_tiles));
    const int tile = static_cast<int>(entry - i * p.by_tiles.d);
    const Kv8Seq sq = kv8_seq(p.seqs, i);
    const int rows = sq.count * static_cast<int>(p.group.d) - tile * p.tile_rows;  // rows left from this tile on
    if (rows <= 0) return;
    const int n_rows = min(rows, p.tile_rows), rho0 = tile * p.tile_rows;
    const int at0 = sq.length - sq.count;
    auto token = [&](int rho) { return static_cast<int>(kv8_div(rho, p.group)); };
    const int pos_lo = at0 + token(rho0), pos_hi = at0 + token(rho0 + n_rows - 1);
    const int key_end = min(pos_hi + 1, sq.length);
    const int page_begin = p.window ? max(pos_lo - p.window + 1, 0) / kKv8Block : 0;
    const int pages = key_end > 0 ? (key_end + kKv8Block - 1) / kKv8Block - page_begin : 0;
    const int active = max(1, min(p.splits, (pages + p.split_pages - 1) / p.split_pages));
    if (split >= active) return;
    const int per = (pages + active - 1) / active;
    const int first = page_begin + min(pages, split * per), last = page_begin + min(pages, (split + 1) * per);
    const int turns = (last - first + kPages - 1) / kPages;
    const bool two = kTiles == 2 && n_rows > 128;  // the streams have different rows; else every other turn each
    auto stream_turns = [&](int stream) { return two ? turns : (turns + 1 - stream) >> 1; };
    auto turn_of = [&](int stream, int n) { return two ? n : 2 * n + stream; };

    const uint32_t s_q = smem_addr(s_mem), s_k = s_q + kTiles * kPlanes * kQBytes, s_v = s_k + kStages * kTileBytes;
    const uint32_t bars = smem_addr(s_bars);
    // by stage of keys and values (turn % kStages), score tile (stream, turn of the stream % 2), and stream
    const uint32_t k_full = bars, v_full = k_full + 8 * kStages, k_empty = v_full + 8 * kStages, v_empty = k_empty + 8 * kStages;
    const uint32_t s_full = v_empty + 8 * kStages, p_full = s_full + 32, o_full = p_full + 16, q_full = o_full + 16, drained = q_full + 8;
    if (threadIdx.x == 0) {
        for (int k = 0; k < kStages; ++k) {
            mbar_init(k_full + 8 * k, kPages);  // pages converted
            mbar_init(v_full + 8 * k, kPages);
            mbar_init(k_empty + 8 * k, two ? 2 : 1);  // tcgen05.commit of the streams that read them
            mbar_init(v_empty + 8 * k, two ? 2 : 1);
            mbar_init(s_full + 8 * k, 1);  // tcgen05.commit: S is there
        }
        for (int k = 0; k < 2; ++k) {
            mbar_init(p_full + 8 * k, 4);  // the stream's warps: the weights are there, the output before has been read
            mbar_init(o_full + 8 * k, 1);  // tcgen05.commit: the output is there, the weights are free
        }
        mbar_init(q_full, 8);
        mbar_init(drained, 1);  // tcgen05.commit: every product that was issued is done
        s_failed = 0;
        s_lo = 255;
        s_hi = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int scale_e = min(max(static_cast<int>(__float_as_uint(p.scale) >> 23) - 127, -126), 126);
    const auto wait = [&](uint32_t bar, int use) {  // the whole warp
        const bool ok = mbar_wait(bar, use & 1, nullptr, &s_failed);
        __syncwarp();
        return ok;
    };
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;  // S [stream][2], then the streams' outputs
    const uint32_t tmem_o = tmem + 4 * kKeys;
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kKv8SoftmaxRegisters));
        // q: four lanes a row
        const int passes = two ? 4 : 2;
        float4 ahead[2][kPieces][2];
        const float unit_scale = p.scale * pow2i(-scale_e), unit_scale_low = p.scale_low * pow2i(-scale_e);
        auto load_q = [&](int pass, float4 (&v)[kPieces][2]) {
            const int rho = rho0 + min((warp * passes + pass) * 8 + (lane & 7), n_rows - 1), at = token(rho);
            const size_t row = static_cast<size_t>(sq.row0 + at) * p.q_stride +
                               static_cast<size_t>(head * p.group.d + rho - at * p.group.d) * D + (lane >> 3) * 8;
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[k][h] = load_row4<kBf16>(p.q, row + k * 32 + h * 4);
        };
        load_q(0, ahead[0]);
        const uint8_t* exps = p.cache.exps + head * 2;
        auto scales_of = [&](int at, bool in) {  // -1: no page
            const int id = in ? sq.pages[at] : -1;
            return static_cast<unsigned>(id) < static_cast<unsigned>(p.cache.pool_pages)
                       ? static_cast<int>(*reinterpret_cast<const unsigned short*>(exps + static_cast<size_t>(id) * p.cache.heads * 2))
                       : -1;
        };
        {  // the split's value scales
            int lo = 255, hi = 0;
            for (int at = first + threadIdx.x; at < last; at += 256) {
                const int ex = scales_of(at, true);
                if (ex >= 0) lo = min(lo, ex >> 8), hi = max(hi, ex >> 8);
            }
            lo = __reduce_min_sync(kFull, lo);
            hi = __reduce_max_sync(kFull, hi);
            if (lane == 0 && lo <= hi) {
                atomicMin(&s_lo, lo);
                atomicMax(&s_hi, hi);
            }
        }
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
            if (pass + 1 < passes) load_q(pass + 1, ahead[1]);
            const int r = (warp * passes + pass) * 8 + (lane & 7);
            const float4(&v)[kPieces][2] = ahead[0];
            uint32_t bits = 0;  // the largest magnitude's; not finite: 0x7f800000 or more
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 x = v[k][h];
                    bits = max(max(max(bits, __float_as_uint(x.x) & 0x7fffffffu), max(__float_as_uint(x.y) & 0x7fffffffu, __float_as_uint(x.z) & 0x7fffffffu)),
                               __float_as_uint(x.w) & 0x7fffffffu);
                }
            bits = max(bits, __shfl_xor_sync(kFull, bits, 8));
            bits = max(bits, __shfl_xor_sync(kFull, bits, 16));
            const bool row_bad = bits >= 0x7f800000u;
            if (row_bad && lane < 8 && r < n_rows) kv8_flag(p.seqs, i, kStatusNonFinite);
            const int e = min(max(static_cast<int>(bits >> 23) - 127, -104), 126);
            // fp32 rows: times the softmax scale (its exponent apart, so that halves hold the products)
            const float up = pow2i(12 - e) * (kBf16 ? 1.0f : unit_scale), up_low = pow2i(12 - e) * unit_scale_low;
            if (lane < 8) s_f[r] = row_bad ? __int_as_float(0x7fc00000) : pow2i(e - 12);  // a bad row's output is NaN
            const uint32_t to = s_q + (r >> 7) * (kPlanes * kQBytes) + (r >> 3 & 15) * kRow8 + (lane >> 3) * 128 + (r & 7) * 16;
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                uint32_t high[4], low[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 x[2] = {make_float2(v[k][h].x, v[k][h].y), make_float2(v[k][h].z, v[k][h].w)};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 y = mul2(x[c], make_float2(up, up));
                        high[2 * h + c] = half2_bits(y.x, y.y);
                        // what the half leaves of the exact product
                        const float2 rest = fma2(x[c], make_float2(up, up), half2_floats(high[2 * h + c] ^ 0x80008000u));
                        const float2 all = fma2(x[c], make_float2(up_low, up_low), rest);
                        low[2 * h + c] = half2_bits(all.x, all.y);
                    }
                }
                kv8_put16(to + k * 512, high[0], high[1], high[2], high[3]);
                if constexpr (!kBf16) kv8_put16(to + k * 512 + kQBytes, low[0], low[1], low[2], low[3]);
            }
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) ahead[0][k][h] = ahead[1][k][h];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const int stream = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, mine = min(two ? stream * 128 + r : r, n_rows - 1);
        const int n_turns = stream_turns(stream);
        // pages that every row of the CTA sees whole: [whole_first, whole_last)
        const int whole_last = max(pos_lo + 1, 0) / kKv8Block;
        const int whole_first = p.window && pos_hi >= p.window ? (pos_hi - p.window) / kKv8Block + 1 : 0;
        // scales of this stream's pages of 8 turns, and of the 8 after them, a lane each
        auto fetch = [&](int n) {
            const int at = first + turn_of(stream, n + lane / kPages) * kPages + lane % kPages;
            return scales_of(at, at < last);
        };
        int scales = fetch(0), scales_next = fetch(8);
        wait(q_full, 0);  // every row's factor, and the value scales' range
        const int ref = s_lo <= s_hi ? kv8_reference(s_lo, s_hi) : 127;  // what eV is relative to
        const auto hide = [&](int ex) { return ex >= 0 && kv8_near((ex >> 8) - ref) ? ex : -1; };  // pages for behind the turns
        scales = hide(scales);
        const float f = s_f[mine] * (kBf16 ? p.scale : pow2i(scale_e));  // of a product of q, as a score
        const int pos = at0 + token(rho0 + mine), low = p.window ? pos - p.window : -1;
        const uint32_t s_tiles = tmem + stream * 2 * kKeys + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t at_o = tmem_o + stream * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t bar_s = s_full + 16 * stream, bar_p = p_full + 8 * stream, bar_o = o_full + 8 * stream;
        float m = -INFINITY, l = 0.0f;
        float o[D];
#pragma unroll
        for (int k = 0; k < D; ++k) o[k] = 0.0f;
        float shrink = 1.0f;  // what O is to be multiplied by before the next output is added
        auto add_output = [&](int n) {
            wait(bar_o, n);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float2 by = make_float2(shrink, shrink);
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float x[32];
                tmem_start(at_o + c, x);
                tmem_arrived(x);
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 z = fma2(make_float2(o[c + k], o[c + k + 1]), by, make_float2(x[k], x[k + 1]));
                    o[c + k] = z.x;
                    o[c + k + 1] = z.y;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        };
        for (int n = 0; n < n_turns; ++n) {
            if (n && n % 8 == 0) {
                scales = hide(scales_next);
                scales_next = fetch(n + 8);
            }
            const int page0 = first + turn_of(stream, n) * kPages, lane0 = n % 8 * kPages;
            const uint32_t at_s = s_tiles + (n & 1) * kKeys;
            // pages of this turn that some row does not see whole, and those that none does: bits
            const unsigned gone = __ballot_sync(kFull, scales < 0) >> lane0 & 0xfu;
            unsigned part = gone;
#pragma unroll
            for (int b = 0; b < kPages; ++b) part |= (page0 + b < whole_first || page0 + b >= whole_last ? 1u : 0u) << b;
            wait(bar_s + 8 * (n & 1), n >> 1);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // positions of chunk c (two pages) that this row sees: bits
            auto seen = [&](int c) {
                const int key = (page0 + 2 * c) * kKv8Block, ahead = pos - key, behind = low - key;  // sees (behind, ahead]
                uint32_t bits = ahead >= 31 ? kFull : ahead < 0 ? 0u : (2u << ahead) - 1;
                if (behind >= 0) bits &= behind >= 31 ? 0u : ~((2u << behind) - 1);
                if (gone >> (2 * c) & 1) bits &= 0xffff0000u;
                if (gone >> (2 * c) & 2) bits &= 0xffffu;
                return bits;
            };
            float top = m;
            const auto largest = [&](float (&x)[32], int c) {
                if (part >> (2 * c) & 3) {
                    const uint32_t bits = seen(c);
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = bits >> k & 1 ? x[k] : -INFINITY;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int ex = __shfl_sync(kFull, scales, lane0 + c * 2 + h);
                    float most = -INFINITY;
#pragma unroll
                    for (int k = h * 16; k < h * 16 + 16; k += 2) most = max3(most, x[k], x[k + 1]);
                    const float u = __int_as_float((ex & 0xff) << 23);
                    const float add = static_cast<float>((ex >> 8) - ref);
                    const float z = fmaf(most, u * f, add);
                    top = fmaxf(top, most == -INFINITY ? -INFINITY : z);
                }
            };
            const auto weigh = [&](float (&x)[32], int c) {
                float less[2];  // 2^-eV
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int ex = __shfl_sync(kFull, scales, lane0 + c * 2 + h);
                    const float u = __int_as_float((ex & 0xff) << 23);
                    const int ev = (ex >> 8) - ref;
                    less[h] = ex < 0 ? 0.0f : pow2i(-ev);
                    const float2 by = make_float2(u * f, u * f);
                    const float2 from = make_float2(static_cast<float>(ev) - top, static_cast<float>(ev) - top);
#pragma unroll
                    for (int k = h * 16; k < h * 16 + 16; k += 2) {
                        const float2 s = make_float2(x[k], x[k + 1]), z = fma2(s, by, from);
                        x[k] = z.x;
                        x[k + 1] = z.y;
                    }
                }
                if (part >> (2 * c) & 3) {
                    const uint32_t bits = seen(c);
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = bits >> k & 1 ? x[k] : -INFINITY;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w_high[8], w_low[8];
                    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int at = h * 16 + (k & 1) * 8 + (k >> 1) * 2;  // the cache's order of positions
                        float2 w = make_float2(ex2(x[at]), ex2(x[at + 1]));
                        sum = add2(sum, w);
                        if constexpr (kBf16) {
                            w_high[k] = half2_bits(w.x, w.y);
                        } else {  // the first 11 bits as they are, and the rest
                            const float2 head = make_float2(__uint_as_float(__float_as_uint(w.x) & 0xffffe000u), __uint_as_float(__float_as_uint(w.y) & 0xffffe000u));
                            w_high[k] = half2_bits(head.x, head.y);
                            w = fma2(head, make_float2(-1.0f, -1.0f), w);
                            w_low[k] = half2_bits(w.x, w.y);
                        }
                    }
                    l = fmaf(sum.x + sum.y, less[h], l);
                    tmem_store8(at_s + c * 32 + h * 8, w_high);
                    if constexpr (!kBf16) tmem_store8(at_s + c * 32 + 16 + h * 8, w_low);
                }
            };
            // A chunk (32 positions) in registers; both of them, from the maximum to the
            // weights, where O leaves the room.
            constexpr bool kHold = D < 128;
            float x[32], y[kHold ? 32 : 1];
            if constexpr (kHold) {
                tmem_start(at_s, x);
                tmem_start(at_s + 32, y);
                tmem_arrived(x);
                tmem_arrived(y);
                largest(x, 0);
                largest(y, 1);
            } else {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    tmem_start(at_s + c * 32, x);
                    tmem_arrived(x);
                    largest(x, c);
                }
            }
            if (!kHold && n) add_output(n - 1);
            const float c = m == top ? 1.0f : ex2(m - top);
            m = top;
            l *= c;
            top = top == -INFINITY ? 0.0f : top - kKv8WeightBits;  // nothing seen yet: weights 0
            if constexpr (kHold) {
                weigh(x, 0);
                if (n) add_output(n - 1);
                weigh(y, 1);
            } else {
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    tmem_start(at_s + c * 32, x);
                    tmem_arrived(x);
                    weigh(x, c);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p);
            shrink = c;
        }
        if (n_turns) add_output(n_turns - 1);
        __syncwarp();
        // The row's share of the result: its sums times what its output or, of a
        // split item, its maximum asks for. Two streams of one row add theirs.
        const auto both_sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        s_ml[stream][r] = make_float2(m, s_failed ? __int_as_float(0x7fc00000) : l);  // a wait that ran out: NaN
        // The streams' products are done, and after a wait that ran out so are those that nobody waited for: the
        // operands' room takes the results.
        if (s_failed)
            for (const long long since = clock64(); !mbar_test(drained, 0) && clock64() - since < kWaitBudgetCycles;) __nanosleep(20);
        both_sync();
        float* s_o = reinterpret_cast<float*>(s_mem) + (stream * 128 + r) * kPitch;
        float most, sum, by;
        const auto factors = [&] {
            const float2 own = s_ml[stream][r], other = s_ml[stream ^ 1][r];
            most = two ? own.x : fmaxf(own.x, other.x);
            const float mine_by = own.x == -INFINITY ? 0.0f : ex2(own.x - most), other_by = two || other.x == -INFINITY ? 0.0f : ex2(other.x - most);
            sum = own.y * (isnan(own.y) ? 1.0f : mine_by) + (two ? 0.0f : other.y * (isnan(other.y) ? 1.0f : other_by));
            by = active == 1 ? mine_by * kv8_inverse(sum, ref, 1.0f) : mine_by;
        };
        factors();
        const bool mixed = s_hi - s_lo > kKv8Spread;  // pages that the turns left out
        const float first_by = mixed ? 1.0f : by;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int g = 0; g < 8; ++g) {  // dims 4g.. of 32 are columns g, 8 + g, 16 + g, 24 + g
                const float2 x = mul2(make_float2(o[j * 32 + g], o[j * 32 + 8 + g]), make_float2(first_by, first_by));
                const float2 y = mul2(make_float2(o[j * 32 + 16 + g], o[j * 32 + 24 + g]), make_float2(first_by, first_by));
                *reinterpret_cast<float4*>(s_o + j * 32 + 4 * g) = make_float4(x.x, x.y, y.x, y.y);
            }
        if (mixed) {  // this row's scores, weights and sums of them in fp32
            const int of = token(rho0 + mine);
            const size_t row = static_cast<size_t>(sq.row0 + of) * p.q_stride + static_cast<size_t>(head * p.group.d + rho0 + mine - of * p.group.d) * D;
#pragma unroll 1
            for (int x = 0; x < n_turns * kPages; ++x) {
                const int page = first + turn_of(stream, x / kPages) * kPages + x % kPages, ex = scales_of(page, page < last);
                if (ex < 0 || kv8_near((ex >> 8) - ref)) continue;
                const uint8_t* block = p.cache.pool + (static_cast<size_t>(sq.pages[page]) * p.cache.heads + head) * (2 * kKv8Block * D);
                float w[kKv8Block];
#pragma unroll
                for (int k = 0; k < kKv8Block; ++k) w[k] = 0.0f;
#pragma unroll 1
                for (int d = 0; d < D; d += 4) {
                    const float4 v = load_row4<kBf16>(p.q, row + d);
#pragma unroll
                    for (int k = 0; k < kKv8Block; ++k) {
                        const uint32_t u = *reinterpret_cast<const uint32_t*>(block + k * D + d);
                        w[k] = fmaf(v.x, kv8_number(u, 0), fmaf(v.y, kv8_number(u, 1), fmaf(v.z, kv8_number(u, 2), fmaf(v.w, kv8_number(u, 3), w[k]))));
                    }
                }
                const float uk = __int_as_float((ex & 0xff) << 23), unit = pow2i((ex >> 8) - ref);
                float now = m;
#pragma unroll
                for (int k = 0; k < kKv8Block; ++k) {
                    const int key = page * kKv8Block + k;
                    w[k] = key <= pos && key > low ? fmaf(w[k] * uk, p.scale, w[k] * uk * p.scale_low) : -INFINITY;
                    now = fmaxf(now, w[k]);
                }
                const float by = m == now ? 1.0f : ex2(m - now), zero = now == -INFINITY ? 0.0f : now - kKv8WeightBits;
                m = now;
                l *= by;
#pragma unroll
                for (int k = 0; k < kKv8Block; ++k) {
                    w[k] = ex2(w[k] - zero);
                    l += w[k];
                    w[k] *= unit;
                }
#pragma unroll 1
                for (int k = 0; k < D / 4; ++k) {
                    float4& at = *reinterpret_cast<float4*>(s_o + 4 * k);
                    float sum[4] = {at.x * by, at.y * by, at.z * by, at.w * by};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {  // positions 2t, 2t + 1, 2t + 8, 2t + 9
                        const uint4 v = *reinterpret_cast<const uint4*>(block + kKv8Block * D + (k * 4 + t) * 16);
                        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            sum[j] = fmaf(w[2 * t], kv8_number(u[j], 0), fmaf(w[2 * t + 1], kv8_number(u[j], 1),
                                     fmaf(w[2 * t + 8], kv8_number(u[j], 2), fmaf(w[2 * t + 9], kv8_number(u[j], 3), sum[j]))));
                    }
                    at = make_float4(sum[0], sum[1], sum[2], sum[3]);
                }
            }
            s_ml[stream][r] = make_float2(m, s_failed ? __int_as_float(0x7fc00000) : l);
            both_sync();
            factors();
            for (int k = 0; k < D; ++k) s_o[k] *= by;
        }
        const size_t part0 = (static_cast<size_t>(item) * p.splits + split) * p.tile_rows;
        if (active > 1 && (two || stream == 0) && stream * 128 + r < n_rows)
            p.part_ml[part0 + stream * 128 + r] = make_float4(most, sum, __int_as_float(ref), 0.0f);
        both_sync();
        if (threadIdx.x == 0 && s_failed) kv8_flag(p.seqs, i, kStatusDevice);
        constexpr int kQuads = D / 4;
        const float* held = reinterpret_cast<const float*>(s_mem);
#pragma unroll 4
        for (int x = threadIdx.x; x < n_rows * kQuads; x += 256) {
            const int row = x / kQuads, d = x % kQuads * 4;
            float4 v = *reinterpret_cast<const float4*>(held + row * kPitch + d);
            if (!two) {
                const float4 w = *reinterpret_cast<const float4*>(held + (128 + row) * kPitch + d);
                v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
            }
            if (active == 1) kv8_store<D, kBf16>(p, sq.row0, rho0 + row, head, d, v);
            else *reinterpret_cast<float4*>(p.part + (part0 + row) * D + d) = v;
        }
        if (active > 1)
            kv8_merge<D, kBf16, 256, 4>(p, 1.0f, both_sync, reinterpret_cast<float4*>(s_mem), &s_last, item, active, p.tile_rows, n_rows,
                                        sq.row0, rho0, head);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kKv8OtherRegisters));
        if (warp < 15) {
            // Pages of keys (unit 8 * turn + page) and of values (unit 8 * turn + 4 + page), every seventh unit.
            const int units = turns * 2 * kPages, converter = warp - 8;
            const int count = units > converter ? (units - converter + kKv8Converters - 1) / kKv8Converters : 0;
            const size_t page_bytes = static_cast<size_t>(p.cache.heads) * 2 * kKv8Block * D;
            const uint8_t* pool = p.cache.pool + static_cast<size_t>(head) * 2 * kKv8Block * D;
            auto fetch_ids = [&](int n) {  // page ids of this warp's units n + lane
                const int unit = converter + (n + lane) * kKv8Converters, at = first + unit / (2 * kPages) * kPages + unit % kPages;
                int id = at < last ? sq.pages[at] : -1;
                if (at < last && static_cast<unsigned>(id) >= static_cast<unsigned>(p.cache.pool_pages)) {
                    kv8_flag(p.seqs, i, kStatusInvalid);
                    id = -1;  // its positions are not seen
                }
                return id;
            };
            // lane 8c + r: 16 dims of key r; lane 8t + g: the cache's piece 4g + t of values. Eight lanes fill a core matrix.
            const int key_row = D == 32 ? lane & 15 : lane & 7, key_piece = D == 32 ? lane >> 4 : lane >> 3;
            const int vg = lane & 7, vt = lane >> 3;
            auto load = [&](uint4 (&w)[kPieces], int n, int id) {
                const int unit = converter + n * kKv8Converters;
                const uint8_t* src = pool + max(id, 0) * page_bytes;
                const bool values = unit & kPages;
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int row = D == 32 ? key_row : (k & 1) * 8 + key_row, piece = D == 32 ? key_piece : (k >> 1) * 4 + key_piece;
                    const int off = values ? kKv8Block * D + k * 512 + (vg * 4 + vt) * 16 : row * D + piece * 16;
                    w[k] = id >= 0 ? *reinterpret_cast<const uint4*>(src + off) : make_uint4(0, 0, 0, 0);
                }
            };
            uint4 a[kPieces], b[kPieces];  // this unit's bytes and the next's
            int ids = fetch_ids(0);
            load(a, 0, __shfl_sync(kFull, ids, 0));
            load(b, 1, __shfl_sync(kFull, ids, 1));
            int ids_next = fetch_ids(32);
            auto convert = [&](const uint4 (&w)[kPieces], int n) {
                const int unit = converter + n * kKv8Converters, turn = unit / (2 * kPages), stage = turn % kStages, page = unit % kPages;
                const bool values = unit & kPages;
                // Units of keys wait for the values' stage too: a warp has a unit of every turn but
                // not of both kinds, and a wait that skipped a phase would take the one before for
                // its own. (P V of the stage's last turn is behind S of this one anyway; units of
                // values do not wait for the keys' stage, which may be two phases on.)
                if (turn >= kStages) {
                    wait(v_empty + 8 * stage, turn / kStages - 1);
                    if (!values) wait(k_empty + 8 * stage, turn / kStages - 1);
                }
                if (values) {
                    const uint32_t to = s_v + stage * kTileBytes + (page * 2 + (vt >> 1)) * 128 + vg * 16 + (vt & 1) * 8;
#pragma unroll
                    for (int k = 0; k < kPieces; ++k) {
                        const uint32_t x[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                        for (int c = 0; c < 4; ++c) kv8_put8(to + (k * 4 + c) * kDim8, kv8_halves<false>(x[c]), kv8_halves<true>(x[c]));
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kPieces; ++k) {
                        const int row = D == 32 ? key_row : (k & 1) * 8 + key_row, piece = D == 32 ? key_piece : (k >> 1) * 4 + key_piece;
                        const uint32_t to = s_k + stage * kTileBytes + (page * 2 + (row >> 3)) * kRow8 + piece * 256 + (row & 7) * 16;
                        kv8_put16(to, kv8_halves<false>(w[k].x), kv8_halves<true>(w[k].x), kv8_halves<false>(w[k].y), kv8_halves<true>(w[k].y));
                        kv8_put16(to + 128, kv8_halves<false>(w[k].z), kv8_halves<true>(w[k].z), kv8_halves<false>(w[k].w),
                                  kv8_halves<true>(w[k].w));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // for the tensor cores
                __syncwarp();
                if (lane == 0) mbar_arrive((values ? v_full : k_full) + 8 * stage);
            };
            for (int n = 0; n < count; n += 2) {
                if (n && n % 32 == 0) {
                    ids = ids_next;
                    ids_next = fetch_ids(n + 32);
                }
                const int ahead = n % 32 + 2;
                convert(a, n);
                load(a, n + 2, __shfl_sync(kFull, ahead < 32 ? ids : ids_next, ahead & 31));
                if (n + 1 < count) convert(b, n + 1);
                load(b, n + 3, __shfl_sync(kFull, ahead < 32 ? ids : ids_next, (ahead + 1) & 31));
            }
        } else {
            constexpr uint32_t idesc_s = umma_idesc_half(128, kKeys), idesc_o = umma_idesc_half(128, D);
            uint32_t leader;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(leader));
            const uint32_t base = __shfl_sync(kFull, tmem, 0);
            const bool apart = __any_sync(kFull, two);
            const int turns0 = __shfl_sync(kFull, stream_turns(0), 0), turns1 = __shfl_sync(kFull, stream_turns(1), 0);
            const uint64_t q_desc = umma_desc_plain(s_q, kRow8), k_desc = umma_desc_plain(s_k, kRow8), v_desc = umma_desc_plain(s_v, kDim8);
            const auto done = [&](uint32_t bar, int use) { return __all_sync(kFull, mbar_test(bar, use & 1)); };
            const auto commit = [&](uint32_t bar) {
                if (leader) umma_commit(bar);
            };
            // A stream's next steps, if what they wait for is there: turns whose S and P V
            // have been issued, and whose P V is known to be done.
            struct Stream {
                int scored, summed, done;
            };
            const auto step = [&](int stream, int n_turns, Stream& at) {
                bool moved = false;
                if (at.done < at.summed && done(o_full + 8 * stream, at.done)) ++at.done;
                if (at.scored < n_turns && at.scored < at.done + 2) {  // S goes where the weights of two turns before lie
                    const int n = at.scored, turn = apart ? n : 2 * n + stream, stage = turn % kStages;
                    if (done(k_full + 8 * stage, turn / kStages)) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t q = q_desc + (apart ? stream : 0) * (kPlanes * kQBytes / 16), k8 = k_desc + stage * (kTileBytes / 16);
#pragma unroll
                        for (int plane = kPlanes - 1; plane >= 0; --plane)
#pragma unroll
                            for (int k = 0; k < D / 16; ++k)
                                umma_half<false>(leader, base + (stream * 2 + (n & 1)) * kKeys, q + plane * (kQBytes / 16) + k * 16, k8 + k * 16,
                                                 idesc_s, plane != kPlanes - 1 || k != 0);
                        commit(s_full + 16 * stream + 8 * (n & 1));
                        commit(k_empty + 8 * stage);
                        ++at.scored;
                        moved = true;
                    }
                }
                if (at.summed < at.scored) {
                    const int n = at.summed, turn = apart ? n : 2 * n + stream, stage = turn % kStages;
                    if (done(p_full + 8 * stream, n) && done(v_full + 8 * stage, turn / kStages)) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t v = v_desc + stage * (kTileBytes / 16);
                        at.done = n;  // the stream has read the output before
#pragma unroll
                        for (int plane = kPlanes - 1; plane >= 0; --plane)
#pragma unroll
                            for (int k = 0; k < kPages; ++k)
                                umma_half<true>(leader, base + 4 * kKeys + stream * 128,
                                                base + (stream * 2 + (n & 1)) * kKeys + (k >> 1) * 32 + plane * 16 + (k & 1) * 8, v + k * 16, idesc_o,
                                                plane != kPlanes - 1 || k != 0);
                        commit(o_full + 8 * stream);
                        commit(v_empty + 8 * stage);
                        ++at.summed;
                        moved = true;
                    }
                }
                return moved;
            };
            Stream s0{0, 0, 0}, s1{0, 0, 0};
            bool ok = __all_sync(kFull, wait(q_full, 0));
            long long since = clock64();
            while (ok && (s0.summed < turns0 || s1.summed < turns1)) {
                bool moved = step(0, turns0, s0);
                moved |= step(1, turns1, s1);
                if (moved) {
                    since = clock64();
                } else if (__any_sync(kFull, *static_cast<volatile int*>(&s_failed) || clock64() - since > kWaitBudgetCycles)) {
                    *static_cast<volatile int*>(&s_failed) = 1;
                    break;
                } else {
                    __nanosleep(20);  // leaves the issue slots to the softmax
                }
            }
            commit(drained);  // no product is on its way when the CTA gives its memory back
            since = clock64();
            while (!done(drained, 0) && !__any_sync(kFull, clock64() - since > kWaitBudgetCycles)) __nanosleep(20);
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 15) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace phonon
