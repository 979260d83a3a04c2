// q8_attn.cu — attention over the 8-bit paged cache: o = sum_j p_j v_j / sum_j p_j with p_j = exp(q.k_j / sqrt(128)), over the
// keys that a query sees (causal, or a sliding window of them), k_j and v_j = code * scale.
//
// This file: single new tokens (decode).  What bounds it is HBM: 264 bytes per key and kv head (two rows of codes, two
// scales), against 4 * 128 * G flops.
//
// Measured (a graph replayed on one state): 64 sessions x 8192 keys, 40 / 8 heads, int8, bf16 activations: 174 us = 6.4 TB/s, 97 % of a
// plain copy (200-213 us = 5.2-5.5 TB/s in calls on three such states in turn); 1 x 131072, int8, fp32: 35-37 us = 3.8 TB/s; 8 x
// (2048-8192), 28 / 4 heads, e4m3, bf16: 20 us; 1 x 1024, int8, fp16: 9.3 us, of which 1.2 are the plan, 0.4 the row, 1.4 q, 0.5 the
// first tile, 0.8 the tiles, 0.9 the partials, 1.6 the gap to the merge, 1.6 the merge.
//
//   * One persistent CTA per SM; the 16-key tiles of all (session, kv group) rows form one line that is dealt out evenly
//     (DecLine); rows that several CTAs worked on are merged by the kernel behind it.
//   * Four producer warps.  Two bring in the codes of K and V with TMA: boxes [128 B][16 slots][kv group], 128-byte swizzle (a row
//     of codes is one swizzle line).  Two load the scales, four keys of a head per lane, and leave what the consumers need
//     of them in shared memory.
//   * Twelve consumer warps: 12 / KVG of them per kv head, each with its own reference maxima, sums and accumulators over
//     every (12 / KVG)-th tile; merged once per row.  Codes become fp16 in registers, exactly, and go to mma.sync m16n8k16 as the
//     16-row operand: S^T = K.Q^T (16 keys x 8 query heads) and O^T += V^T.P^T (16 dims x 8 heads), so that none of the
//     instruction's rows is padding but for the heads beyond G.  A lane reads 32 consecutive codes of a key: the
//     contraction index may be permuted freely as long as q's fragments follow.  V needs pairs of keys side by side: bytes are
//     interleaved with permutes, and the rows of product j are the dims 16 g + 2 j (+ 1).  P goes from the accumulator layout to
//     the operand layout with movmatrix.
//   * int8 K with q in one part: the byte code + 128 is taken as an fp16 subnormal, (code + 128) 2^-24, which costs no arithmetic; the
//     accumulators start at -128 2^-24 sum(q).  What the offset's size takes from the accumulators' bits stays below what rounding q to
//     fp16 does.  With q in two parts it would not (keys of small codes beside a large one, queries of one sign: 2^-15 of sum |q k|
//     instead of 2^-21), so there the codes go in as they are, one subtraction a pair.  (Nor for V: there the offset would be a sum of
//     weights, hundreds of times the result.)
//   * fp32 and fp16 activations: q and p as fp16 hi + lo, two instructions each, so that outputs are as good as fp32 arithmetic gives
//     them (rounded once, fp16 outputs would be 5e-4 off instead of 2e-4).  bf16 activations: q (rotated) and p rounded to fp16,
//     which bf16's own 2^-9 hides.
//   * The scale of K multiplies the finished score.  The scale of V goes into the exponent: w_j = 2^(x_j + log2 sv_j - ref), so
//     the weights that multiply the codes stay inside fp16's range whatever the scales are; the softmax sum adds w_j / sv_j.
#include "q8_common.cuh"

namespace novab {
namespace {

constexpr int kSetupTiles = 8;       // work-split weight of starting a row inside a CTA, in tiles (8 x (2k-8k): 2 22.6 us, 4 22.4, 8 20.8, 12 22.5)
constexpr int kDecRows = 512;        // (session, kv group) rows of a launch
constexpr int kMinTiles = 4;         // a CTA gets at least that many tiles (fewer partial rows to merge for short contexts)

template <int KVG>
struct DecCfg {
    static constexpr int kCons = 12;                        // consumer warps; with four producers 16, which leave 128 registers a thread
    static constexpr int kSub = kCons / KVG;                // ... per kv head
    static constexpr int kStages = 36 / KVG;                // 144 KiB of tiles in flight; a stage always goes to the same warps
    static constexpr int kHalf = KVG * 2048;                // K (or V) codes of a tile
    static constexpr int kTile = 2 * kHalf;
    static constexpr int kScales = KVG * 192;               // K scales | logarithms of V's | reciprocals of V's
    static constexpr int kMergeFloats = KVG * kSub * 36 * 32;
    static constexpr int kRawSteps = 8;                     // rings of raw scales (K, V), steps of 512 bytes
    static constexpr int kSmem = kStages * (kTile + kScales) + 2 * kRawSteps * 512 + kMergeFloats * 4 + 1024;
    static constexpr int kThreads = 32 * (kCons + 4);
    static constexpr int kBatch = 8 / KVG;                  // tiles that a producer of codes issues at a time
    static_assert(kStages % kSub == 0, "stages and consumer warps");
};

// The line of work: per (session, group) row kSetupTiles and its tiles (a row without a new token: nothing), in 32 bits, cut off
// where it would pass them.
struct DecPlan {
    int prefix[kDecRows + 1];
    int keys[kDecRows];
    int row[kDecRows];
    int slice[kDecRows];
};

__device__ __forceinline__ int dec_low(const Q8Launch& a, int keys) { return a.window > 0 && keys > a.window ? keys - a.window : 0; }      // first key that is seen
__device__ __forceinline__ int dec_first_tile(const Q8Launch& a, int keys) { return dec_low(a, keys) >> 4; }

// Tiles of a row: keys behind the block table are not looked for, but there is always one tile.
__device__ __forceinline__ int dec_tiles(const Q8Launch& a, int keys) {
    const int end = keys < a.keys_cap ? keys : a.keys_cap;
    return max(((end + 15) >> 4) - dec_first_tile(a, keys), 1);
}

__device__ __forceinline__ int dec_setup(int row) { return row > 0 ? kSetupTiles : 0; }

__device__ inline void dec_build_plan(const Q8Launch& a, DecPlan& p, int n_groups, bool flag) {
    for (int s = (int)threadIdx.x; s < a.n_sessions; s += (int)blockDim.x) {      // (all loads at once: one trip to memory)
        int first, count;
        q8_rows(a, s, first, count);
        const int pos = __ldg(a.n_past + s), slice = a.slice_ids ? __ldg(a.slice_ids + s) : s;
        int keys = 0;
        if (count > 0) {
            if (pos < 0 || pos >= kQ8MaxPos || (a.rope_cs && pos >= a.rope_rows)) {
                if (flag) q8_flag(a, NOVA_ERR_INVALID);
            } else {
                keys = pos + 1;
                if (flag && keys > a.keys_cap) q8_flag(a, NOVA_ERR_BAD_TABLE);
            }
        }
        p.keys[s] = keys;
        p.row[s] = first;
        p.slice[s] = slice;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = (int)threadIdx.x, rows = a.n_sessions * n_groups;
        uint32_t carry = 0;
        if (lane == 0) p.prefix[0] = 0;
        for (int base = 0; base < rows; base += 32) {
            const int r = base + lane, keys = r < rows ? p.keys[r / n_groups] : 0;
            uint32_t v = keys > 0 ? (uint32_t)(dec_tiles(a, keys) + dec_setup(r)) : 0u;
            v = min(v, 0x7ffffffu);                            // (the sum of 32 stays inside 32 bits)
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += t;
            }
            const uint32_t sum = min(carry + min(v, 0x7fffffffu), 0x7fffffffu);
            if (r < rows) p.prefix[r + 1] = (int)sum;
            carry = __shfl_sync(0xffffffffu, sum, 31);
        }
        if (flag && lane == 0 && carry == 0x7fffffffu) q8_flag(a, NOVA_ERR_INVALID);
    }
    __syncthreads();
}

// The line dealt out evenly: the first `extra` CTAs get per + 1 entries, the others per.
struct DecLine {
    int rows, n_groups, total, n_ctas, per, extra;
    __device__ __forceinline__ int begin(int c) const { return c * per + min(c, extra); }
    __device__ __forceinline__ int owner(int t) const {
        const int wide = extra * (per + 1);
        return t < wide ? t / (per + 1) : extra + (t - wide) / per;
    }
};
__device__ __forceinline__ DecLine dec_line(const Q8Launch& a, const DecPlan& p, int n_groups, int grid) {
    DecLine ln;
    ln.rows = a.n_sessions * n_groups;
    ln.n_groups = n_groups;
    ln.total = p.prefix[ln.rows];
    const int most = ln.total / kMinTiles + (ln.total % kMinTiles != 0);
    ln.n_ctas = most < grid ? most : grid;
    ln.per = ln.total > 0 ? ln.total / ln.n_ctas : 0;
    ln.extra = ln.total - ln.per * ln.n_ctas;
    return ln;
}

// What a CTA does of one row: from entry pos of the line to the row's end or hi.  By whole warps.
struct DecSegment {
    int row, session, group;
    int first, count;      // tiles, counted from the row's first
    int span;              // entries of the line
    bool whole;            // no other CTA works on the row
};
__device__ __forceinline__ DecSegment dec_segment(const DecPlan& p, const DecLine& ln, int pos, int lo, int hi) {
    const int lane = (int)threadIdx.x & 31, stride = (ln.rows + 31) >> 5;
    // the last row that begins at pos or before (rows without work begin where the next one does)
    int at = lane * stride;
    int row = (__popc(__ballot_sync(0xffffffffu, at < ln.rows && p.prefix[at] <= pos)) - 1) * stride;
    if (stride > 1) {
        at = row + lane;
        row += __popc(__ballot_sync(0xffffffffu, lane < stride && at < ln.rows && p.prefix[at] <= pos)) - 1;
    }
    DecSegment sg;
    const int begin = p.prefix[row], row_end = p.prefix[row + 1], end = row_end < hi ? row_end : hi;
    sg.row = row;
    sg.session = row / ln.n_groups;
    sg.group = row - sg.session * ln.n_groups;
    sg.span = end - pos;
    sg.first = max(pos - begin - dec_setup(row), 0);
    sg.count = max(end - begin - dec_setup(row), 0) - sg.first;
    sg.whole = begin >= lo && row_end <= hi;
    return sg;
}

// A CTA that has given up on a wait stays for a millisecond more: copies that it has on their way land in microseconds, and none may when
// its shared memory is another's.
__device__ __forceinline__ void dec_settle(const volatile int* aborted) {
    if (!*aborted) return;
    const unsigned long long t0 = now_ns();
    for (int i = 0; i < 100000 && now_ns() - t0 < 1000000ull; ++i) __nanosleep(1000);
}

// kLo: q and p in two fp16 parts (fp32 and fp16 activations, unless one_part)
template <int KVG, int kFmt, bool kLo>
__global__ void __launch_bounds__(DecCfg<KVG>::kThreads, 1)
q8_decode_kernel(Q8Launch a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    using Cfg = DecCfg<KVG>;
    constexpr int kStages = Cfg::kStages, kSub = Cfg::kSub;
    extern __shared__ unsigned char smem_raw[];
    __shared__ DecPlan s_plan;
    __shared__ __align__(8) unsigned long long s_full[kStages];
    __shared__ __align__(8) unsigned long long s_empty[kStages];
    __shared__ uint32_t s_mask[kStages];      // which of the tile's 16 keys count
    __shared__ int s_phys[kStages];           // the page of the tile's last key (where a new token goes)
    __shared__ int s_abort;

    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const int G = a.n_heads / a.n_kv_heads, n_groups = a.n_kv_heads / KVG;
    const int heads_per_row = KVG * G;
    const uint32_t tile0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t scale0 = tile0 + kStages * Cfg::kTile;
    float* const merge = reinterpret_cast<float*>(smem_raw + (scale0 - smem_u32(smem_raw)) + kStages * Cfg::kScales + 2 * Cfg::kRawSteps * 512);
    // the operands are q / 8 (rotated fp16 values stay inside fp16) and codes, those of int8 K, with q in one part, plus 128 and times 2^-24
    constexpr bool kOffset = kFmt == NOVA_KV_I8 && !kLo;
    constexpr float kToLog2 = kAttnScale * kLog2e * 8.f * (kOffset ? 16777216.f : 1.f);
    // a page of 8 tokens is half a tile: two boxes of 8 slots, [half][kv head][8]; otherwise [kv head][16]
    const bool p8 = a.kv_shift == 3;
    const uint32_t head_step = p8 ? 1024u : 2048u, half_step = p8 ? KVG * 1024u : 1024u;

    if (threadIdx.x == 32 * Cfg::kCons) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 4);        // codes and scales of K and V
            mbar_init(smem_u32(&s_empty[i]), KVG);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmk) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmv) : "memory");
    }
    // Nothing of the caller's is read before the kernels before this one are done; the merge kernel, which reads positions and
    // row starts before its own wait, is let go only then.
    pdl_wait();
    pdl_launch_dependents();
    dec_build_plan(a, s_plan, n_groups, blockIdx.x == 0);
    const DecLine ln = dec_line(a, s_plan, n_groups, (int)gridDim.x);
    if ((int)blockIdx.x >= ln.n_ctas) return;
    const int lo = ln.begin((int)blockIdx.x), hi = ln.begin((int)blockIdx.x + 1);

    // ------------------------------------------------------------------------------------------------ producers
    // Each of the four goes through ALL tiles in order: a stage's fill waits for the release of the fill before, which the same
    // warp has taken part in, so a parity is never taken for the one two fills ago.
    const int tpp = a.kv_shift > 4 ? a.kv_shift - 4 : 0;               // log2(tiles per page)
    // entries of the block table behind tile i of a segment (the second: 8-token pages); -1: a bad one, -2: nothing to bring (no key of
    // the page is there, or none is in the window: an 8-token page in front of one that is, whose entry may be gone)
    auto fetch = [&](const int32_t* table, int keys, int low, int t, bool real, int& e0, int& e1) {
        auto entry = [&](int64_t page, int first_key) -> int {
            if (first_key >= keys || (p8 && first_key + 8 <= low)) return -2;
            if (page >= a.table_stride) return -1;
            const int e = __ldg(table + page);
            return e >= 0 && e < a.nb ? e : -1;
        };
        e0 = e1 = -2;
        if (!real) return;
        if (p8) {
            e0 = entry(2 * (int64_t)t, 16 * t);
            e1 = entry(2 * (int64_t)t + 1, 16 * t + 8);
        } else {
            e0 = entry(t >> tpp, 16 * t);
        }
    };
    if (warp < Cfg::kCons + 2 && warp >= Cfg::kCons) {
        // Codes of K and of V, a batch of tiles at a time, one lane per tile: what a copy costs its thread (wait, byte count,
        // issue: several hundred cycles) is then paid once per batch.  A batch waits for all its stages, so it is a small part of the
        // ring: the rest stays in flight meanwhile.
        const bool is_v = warp == Cfg::kCons + 1;
        const unsigned long long policy = l2_policy_evict_first();
        const CUtensorMap* const tm = is_v ? &tmv : &tmk;
        const int row0 = (a.layer * a.nb) << a.kv_shift;
        uint32_t it0 = 0;                                                   // tiles before this segment
        for (int pos = lo; pos < hi;) {
            const DecSegment sg = dec_segment(s_plan, ln, pos, lo, hi);
            pos += sg.span;
            const int keys = s_plan.keys[sg.session];
            const int t0 = dec_first_tile(a, keys) + sg.first, low = dec_low(a, keys);
            const int32_t* table = a.tables + (int64_t)s_plan.slice[sg.session] * a.table_stride;
            int n0, n1, c0 = 0, c1 = 0;
            fetch(table, keys, low, t0 + lane, lane < sg.count, n0, n1);
            uint32_t stage = (it0 + (uint32_t)lane) % kStages, round = (it0 + (uint32_t)lane) / kStages;
#pragma unroll 1
            for (int b = 0; b < sg.count; b += Cfg::kBatch) {
                if ((b & 31) == 0) {                                        // 32 entries at a time, the next 32 on their way
                    c0 = n0;
                    c1 = n1;
                    const int nx = b + 32 + lane;
                    fetch(table, keys, low, t0 + nx, nx < sg.count, n0, n1);
                }
                const int i = b + lane, t = t0 + i;
                const int e0 = __shfl_sync(0xffffffffu, c0, i & 31);
                int e1 = -2;
                if (p8) e1 = __shfl_sync(0xffffffffu, c1, i & 31);
                const bool mine = lane < Cfg::kBatch && i < sg.count;
                const bool free = !mine || round == 0 || mbar_wait(smem_u32(&s_empty[stage]), (round - 1) & 1, &s_abort);
                if (!__all_sync(0xffffffffu, free)) {
                    if (lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);
                    dec_settle(&s_abort);
                    return;
                }
                if (mine) {
                    const uint32_t bar = smem_u32(&s_full[stage]);
                    const uint32_t dst = tile0 + stage * Cfg::kTile + (is_v ? (uint32_t)Cfg::kHalf : 0u);
                    const int slot = p8 ? 0 : (t << 4) & ((1 << a.kv_shift) - 1);
                    const uint32_t halves = (uint32_t)(p8 ? (e0 >= 0) + (e1 >= 0) : 2 * (e0 >= 0));
                    if (!is_v) {
                        if (e0 == -1 || e1 == -1) q8_flag(a, NOVA_ERR_BAD_TABLE);
                        uint32_t mask = p8 ? (e0 >= 0 ? 0xffu : 0u) | (e1 >= 0 ? 0xff00u : 0u) : (e0 >= 0 ? 0xffffu : 0u);
                        if (keys - 16 * t < 16) mask &= (1u << (keys - 16 * t)) - 1u;
                        if (low > 16 * t) mask &= ~((1u << (low - 16 * t < 16 ? low - 16 * t : 16)) - 1u);
                        s_mask[stage] = mask;
                        s_phys[stage] = p8 && e1 >= 0 ? e1 : e0;
                    }
                    if (halves) mbar_expect_tx(bar, halves * (uint32_t)(Cfg::kHalf / 2));
                    else mbar_arrive(bar);
                    if (e0 >= 0) tma_load_3d_hint(dst, tm, 0, row0 + (e0 << a.kv_shift) + slot, sg.group * KVG, bar, policy);
                    if (p8 && e1 >= 0) tma_load_3d_hint(dst + half_step, tm, 0, row0 + (e1 << a.kv_shift), sg.group * KVG, bar, policy);
                }
                __syncwarp();
                stage += Cfg::kBatch;
                if (stage >= kStages) {
                    stage -= kStages;
                    ++round;
                }
            }
            it0 += (uint32_t)sg.count;
        }
        return;
    }
    if (warp >= Cfg::kCons + 2) {
        // Scales of K and of V: a lane takes four keys of one head of a tile, 8 / KVG tiles at a time, and leaves what the consumers
        // multiply with: K's scale times 1/sqrt(128) log2 e (and what the operands were scaled by), V's logarithm and reciprocal.
        // The raw scales arrive (cp.async) in a ring of the warp's own, far enough ahead of their use: they are short runs all over
        // the pools, about 2 us away when HBM is busy.
        constexpr int kPer = 8 / KVG, kDepth = Cfg::kRawSteps - 1;           // tiles of a step (512 bytes of scales); steps ahead
        const bool is_v = warp == Cfg::kCons + 3;
        const int sub_tile = lane / (4 * KVG), quad = lane & 3, h = (lane >> 2) % KVG;
        const uint32_t raw0 = scale0 + kStages * Cfg::kScales + (uint32_t)(is_v ? Cfg::kRawSteps * 512 : 0) + (uint32_t)lane * 16u;
        const uint32_t dst0 = scale0 + (uint32_t)((is_v ? KVG * 64 : 0) + h * 64 + quad * 16);
        const int slot_mask = p8 ? 0 : (1 << a.kv_shift) - 1, slot_add = p8 ? 4 * (quad & 1) : 4 * quad;
        uint32_t it0 = 0;
        for (int pos = lo; pos < hi;) {
            const DecSegment sg = dec_segment(s_plan, ln, pos, lo, hi);
            pos += sg.span;
            const int keys = s_plan.keys[sg.session], t0 = dec_first_tile(a, keys) + sg.first, low = dec_low(a, keys);
            const int32_t* table = a.tables + (int64_t)s_plan.slice[sg.session] * a.table_stride;
            const float* const mine0 = (is_v ? a.scale_v : a.scale_k) + ((((int64_t)a.layer * a.nb) * a.n_kv_heads + sg.group * KVG + h) << a.kv_shift);
            const int steps = (sg.count + kPer - 1) / kPer;
            int n0, n1, c0 = 0, c1 = 0;
            fetch(table, keys, low, t0 + lane, lane < sg.count, n0, n1);
            uint32_t stage = (it0 + (uint32_t)sub_tile) % kStages, round = (it0 + (uint32_t)sub_tile) / kStages;
            int i = sub_tile - kDepth * kPer;                               // the tile that this step converts
#pragma unroll 1
            for (int step = 0; step < steps + kDepth; ++step, i += kPer) {
                if (step < steps) {
                    const int f = step * kPer;
                    if ((f & 31) == 0) {                                    // 32 entries at a time, the next 32 on their way
                        c0 = n0;
                        c1 = n1;
                        const int nx = f + 32 + lane;
                        fetch(table, keys, low, t0 + nx, nx < sg.count, n0, n1);
                    }
                    int e = __shfl_sync(0xffffffffu, c0, (f + sub_tile) & 31);       // (below 0 behind the segment's last tile too)
                    if (p8) {
                        const int f1 = __shfl_sync(0xffffffffu, c1, (f + sub_tile) & 31);
                        if (quad >= 2) e = f1;
                    }
                    const int slot = (((t0 + f + sub_tile) << 4) & slot_mask) + slot_add;
                    const uint32_t raw = raw0 + (uint32_t)(step & (Cfg::kRawSteps - 1)) * 512u;
                    if (e >= 0) cp_async16(raw, mine0 + (((int64_t)e * a.n_kv_heads) << a.kv_shift) + slot);
                    else sts128(raw, make_float4(0.f, 0.f, 0.f, 0.f));
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (step < kDepth) continue;
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth) : "memory");
                const bool mine = i < sg.count;                        // a lane converts what it has brought itself
                const uint4 u = lds128(raw0 + (uint32_t)((step - kDepth) & (Cfg::kRawSteps - 1)) * 512u);
                const float4 v = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
                const bool free = !mine || round == 0 || mbar_wait(smem_u32(&s_empty[stage]), (round - 1) & 1, &s_abort);
                if (!__all_sync(0xffffffffu, free)) {
                    if (lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);
                    break;
                }
                const uint32_t dst = dst0 + stage * Cfg::kScales;
                if (mine) {
                    if (!is_v) {
                        sts128(dst, make_float4(v.x * kToLog2, v.y * kToLog2, v.z * kToLog2, v.w * kToLog2));
                    } else {
                        auto at_least = [](float x) { return x < kQ8MinScale ? kQ8MinScale : x; };      // (a NaN stays one)
                        const float4 m = make_float4(at_least(v.x), at_least(v.y), at_least(v.z), at_least(v.w));
                        sts128(dst, make_float4(lg2(m.x), lg2(m.y), lg2(m.z), lg2(m.w)));
                        sts128(dst + KVG * 64, make_float4(rcp(m.x), rcp(m.y), rcp(m.z), rcp(m.w)));
                    }
                }
                __syncwarp();
                if (mine && lane % (4 * KVG) == 0) mbar_arrive(smem_u32(&s_full[stage]));
                stage += kPer;
                if (stage >= kStages) {
                    stage -= kStages;
                    ++round;
                }
            }
            it0 += (uint32_t)sg.count;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }

    // ------------------------------------------------------------------------------------------------ consumers
    const int w = warp % KVG, sub = warp / KVG;       // kv head of the group, which of its warps
    const int g = lane >> 2, t = lane & 3;
    uint32_t it = 0;                                  // tiles of the segments before
    int stage = sub;                                  // of this warp's next tile, and the parity of its fill
    uint32_t parity = 0;
    for (int pos = lo; pos < hi;) {
        const DecSegment sg = dec_segment(s_plan, ln, pos, lo, hi);
        pos += sg.span;
        const int s = sg.session, kvh = sg.group * KVG + w;
        const int keys = s_plan.keys[s], row = s_plan.row[s], t0 = dec_first_tile(a, keys) + sg.first;

        // q of the kv head's query heads: its warps rotate, scale and round them together, 8 dims a thread, and leave them in shared
        // memory (each warp for itself took 2 us instead of 1: all of them would do the same work); then a lane takes head g's
        // dims 32 t .. 32 t + 31, four per contraction step.  Row of a head: its 16-byte chunk 4 t + k at place 4 k + t, xor 4 in
        // odd rows, so that the fragments' loads meet no bank twice.
        uint32_t qh[8][2], ql[kLo ? 8 : 1][2];
        float off0 = 0.f, off1 = 0.f;             // what the accumulators of heads 2 t and 2 t + 1 start at
        {
            const uint32_t stash = smem_u32(merge) + (uint32_t)w * kSub * 36u * 128u;       // [8][256] fp16, its second part, [8] sums
#pragma unroll 1
            for (int un = 32 * sub + lane; un < 16 * G + (16 * G & 16); un += 32 * kSub) {  // (whole warps)
                const int hd = un >> 4, i = un & 15;
                const bool real = hd < G;
                const int d0 = a.neox || !a.rope_cs ? 4 * i : 8 * i, d1 = a.neox || !a.rope_cs ? 64 + 4 * i : 8 * i + 4;
                float4 x0 = make_float4(0.f, 0.f, 0.f, 0.f), x1 = x0, c = x0, n = x0;
                if (real) {
                    const int64_t qe = (int64_t)row * a.q_stride + (int64_t)(kvh * G + hd) * kHeadDim;
                    if (a.rope_cs) {
                        c = __ldg(reinterpret_cast<const float4*>(a.rope_cs + (int64_t)(keys - 1) * 64) + i);
                        n = __ldg(reinterpret_cast<const float4*>(a.rope_sn + (int64_t)(keys - 1) * 64) + i);
                    }
                    x0 = q8_load4(a.q, qe + d0, a.io);
                    x1 = q8_load4(a.q, qe + d1, a.io);
                }
                if (a.rope_cs) {
                    float4 u, v;
                    if (a.neox) {
                        u = make_float4(__fmaf_rn(x0.x, c.x, -__fmul_rn(x1.x, n.x)), __fmaf_rn(x0.y, c.y, -__fmul_rn(x1.y, n.y)),
                                        __fmaf_rn(x0.z, c.z, -__fmul_rn(x1.z, n.z)), __fmaf_rn(x0.w, c.w, -__fmul_rn(x1.w, n.w)));
                        v = make_float4(__fmaf_rn(x0.x, n.x, __fmul_rn(x1.x, c.x)), __fmaf_rn(x0.y, n.y, __fmul_rn(x1.y, c.y)),
                                        __fmaf_rn(x0.z, n.z, __fmul_rn(x1.z, c.z)), __fmaf_rn(x0.w, n.w, __fmul_rn(x1.w, c.w)));
                    } else {
                        u = make_float4(__fmaf_rn(x0.x, c.x, -__fmul_rn(x0.y, n.x)), __fmaf_rn(x0.x, n.x, __fmul_rn(x0.y, c.x)),
                                        __fmaf_rn(x0.z, c.y, -__fmul_rn(x0.w, n.y)), __fmaf_rn(x0.z, n.y, __fmul_rn(x0.w, c.y)));
                        v = make_float4(__fmaf_rn(x1.x, c.z, -__fmul_rn(x1.y, n.z)), __fmaf_rn(x1.x, n.z, __fmul_rn(x1.y, c.z)),
                                        __fmaf_rn(x1.z, c.w, -__fmul_rn(x1.w, n.w)), __fmaf_rn(x1.z, n.w, __fmul_rn(x1.w, c.w)));
                    }
                    x0 = u;
                    x1 = v;
                }
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float4 x = e ? x1 : x0;
                    const float f[4] = {x.x * 0.125f, x.y * 0.125f, x.z * 0.125f, x.w * 0.125f};
                    const __half2 h0 = __floats2half2_rn(f[0], f[1]), h1 = __floats2half2_rn(f[2], f[3]);
                    const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                    const int d = e ? d1 : d0, chunk = d >> 3;
                    const uint32_t dst = stash + (uint32_t)hd * 256u + (uint32_t)(((4 * (chunk & 3) + (chunk >> 2)) ^ (4 * (hd & 1))) * 16 + (d & 4) * 2);
                    sum += (b0.x + b0.y) + (b1.x + b1.y);
                    if (real) {
                        sts64(dst, *reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                        if constexpr (kLo) sts64(dst + 2048u, pack_h2(f[0] - b0.x, f[1] - b0.y), pack_h2(f[2] - b1.x, f[3] - b1.y));
                    }
                }
                if constexpr (kOffset) {
#pragma unroll
                    for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (real && i == 0) sts_f1(stash + 4096u + (uint32_t)hd * 4u, sum);
                }
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t src = stash + (uint32_t)g * 256u + (uint32_t)(((4 * k + t) ^ (4 * (g & 1))) * 16);
                const uint4 h = g < G ? lds128(src) : make_uint4(0u, 0u, 0u, 0u);
                qh[2 * k][0] = h.x, qh[2 * k][1] = h.y, qh[2 * k + 1][0] = h.z, qh[2 * k + 1][1] = h.w;
                if constexpr (kLo) {
                    const uint4 l = g < G ? lds128(src + 2048u) : make_uint4(0u, 0u, 0u, 0u);
                    ql[2 * k][0] = l.x, ql[2 * k][1] = l.y, ql[2 * k + 1][0] = l.z, ql[2 * k + 1][1] = l.w;
                }
            }
            if constexpr (kOffset) {                                                                // 128 * 2^-24
                if (2 * t < G) off0 = -7.62939453125e-06f * lds_f1(stash + 4096u + 8u * t);
                if (2 * t + 1 < G) off1 = -7.62939453125e-06f * lds_f1(stash + 4096u + 8u * t + 4u);
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");               // (the merge uses the same place)
        }
        // heads 2 t and 2 t + 1: reference maximum (log2 units), this lane's share of the sum, dims 16 g .. 16 g + 15
        float ref0 = -INFINITY, ref1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        float o[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

        const uint32_t it_end = it + (uint32_t)sg.count;
        for (uint32_t i = it + (((uint32_t)sub + kSub - it % kSub) % kSub); i < it_end; i += kSub) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[stage]), parity, &s_abort))) {
                if (lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);      // the result is void; the warp still meets its siblings below
                break;
            }
            const uint32_t mask = s_mask[stage];
            const uint32_t sk = tile0 + (uint32_t)stage * Cfg::kTile + w * head_step, sv = sk + Cfg::kHalf;
            const uint32_t ck = scale0 + (uint32_t)stage * Cfg::kScales + w * 64u;
            const int tile = t0 + (int)(i - it);
            bool patched = false;
            if (a.append && tile == (keys - 1) >> 4 && (mask >> ((keys - 1) & 15) & 1)) {
                // this tile takes the new token: rotate, quantise, write it into the pool and into the staged copy
                patched = true;
                const int slot = (keys - 1) & 15;
                const int64_t page = (int64_t)a.layer * a.nb + s_phys[stage];
                const int pslot = (keys - 1) & ((1 << a.kv_shift) - 1);
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2) {
                    float4 x = q8_load4(i2 ? a.v : a.k, (int64_t)row * (i2 ? a.v_stride : a.k_stride) + (int64_t)kvh * kHeadDim + 4 * lane, a.io);
                    if (!i2 && a.rope_cs) {
                        x = q8_rotate(x, keys - 1, lane, a);
                        if (a.k_rot) *reinterpret_cast<float4*>(a.k_rot + ((int64_t)row * a.n_kv_heads + kvh) * kHeadDim + 4 * lane) = x;
                    }
                    const float amax = fmaxf(q8_amax(x), kQ8MinAmax);
                    const float inv = __fdiv_rn(q8_qmax<kFmt>(), amax), scale = __fdiv_rn(amax, q8_qmax<kFmt>());
                    const uint32_t code = q8_encode4<kFmt>(make_float4(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv)));
                    *reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(i2 ? a.pool_v : a.pool_k) +
                                                 (((page << a.kv_shift) + pslot) * a.n_kv_heads + kvh) * kHeadDim + 4 * lane) = code;
                    const uint32_t dst = (i2 ? sv : sk) + (slot >> 3) * half_step + (slot & 7) * 128u + ((((uint32_t)lane >> 2) ^ (slot & 7)) << 4) + ((lane & 3) << 2);
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(code) : "memory");
                    if (lane == 0) {
                        (i2 ? a.scale_v : a.scale_k)[((page * a.n_kv_heads + kvh) << a.kv_shift) + pslot] = scale;
                        sts_f1(ck + (i2 ? KVG * 64u : 0u) + slot * 4u, i2 ? lg2(scale) : scale * kToLog2);
                        if (i2) sts_f1(ck + KVG * 128u + slot * 4u, rcp(scale));
                    }
                }
                __syncwarp();
            }
            if (mask) {
                // Everything of the tile into registers, so that the stage can be filled again while the rest is computed: codes 32 t ..
                // of keys g and g + 8 (two swizzled 16-byte pieces each), codes 16 g .. of keys 2t, 2t + 1, 2t + 8, 2t + 9, scales.
                uint4 kw[2][2], vw[4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    kw[half][0] = lds128(sk + g * 128u + (((2 * t + half) ^ g) << 4));
                    kw[half][1] = lds128(sk + half_step + g * 128u + (((2 * t + half) ^ g) << 4));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) vw[e] = lds128(sv + (e >> 1) * half_step + (2 * t + (e & 1)) * 128u + ((g ^ (2 * t + (e & 1))) << 4));
                const float ka = lds_f1(ck + 4 * g), kb = lds_f1(ck + 4 * g + 32), la = lds_f1(ck + KVG * 64 + 4 * g), lb = lds_f1(ck + KVG * 64 + 4 * g + 32);
                float ra = lds_f1(ck + KVG * 128 + 4 * g), rb = lds_f1(ck + KVG * 128 + 4 * g + 32);
                if (patched) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
                // S^T = K.Q^T
                float c[4] = {off0, off1, off0, off1};
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint4 wa = kw[ks >> 2][0], wb = kw[ks >> 2][1];
                    const int k4 = ks & 3;
                    uint32_t a0, a1, a2, a3;
                    const uint32_t w0 = k4 == 0 ? wa.x : k4 == 1 ? wa.y : k4 == 2 ? wa.z : wa.w, w1 = k4 == 0 ? wb.x : k4 == 1 ? wb.y : k4 == 2 ? wb.z : wb.w;
                    if constexpr (kOffset) {
                        q8_k_to_h2(w0, a0, a2);
                        q8_k_to_h2(w1, a1, a3);
                    } else {
                        q8_to_h2<kFmt>(w0, a0, a2);
                        q8_to_h2<kFmt>(w1, a1, a3);
                    }
                    mma_full(c, a0, a1, a2, a3, qh[ks][0], qh[ks][1]);
                    if constexpr (kLo) mma_full(c, a0, a1, a2, a3, ql[ks][0], ql[ks][1]);
                }
                // x[e]: keys g (e = 0, 1) and g + 8 (e = 2, 3), heads 2 t and 2 t + 1
                float x[4] = {fmaf(c[0], ka, la), fmaf(c[1], ka, la), fmaf(c[2], kb, lb), fmaf(c[3], kb, lb)};
                if (mask != 0xffffu) {             // what is masked may hold anything
                    if (!((mask >> g) & 1)) {
                        x[0] = x[1] = -INFINITY;
                        ra = 0.f;
                    }
                    if (!((mask >> (g + 8)) & 1)) {
                        x[2] = x[3] = -INFINITY;
                        rb = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((mask >> (2 * t + (e & 1) + 8 * (e >> 1))) & 1)) vw[e] = make_uint4(0u, 0u, 0u, 0u);
                }
                // (2^kQ8Top cancels between the outputs and l)
                float m0 = fmaxf(x[0], x[2]), m1 = fmaxf(x[1], x[3]);
                if (__any_sync(0xffffffffu, m0 > ref0 + kQ8Step || m1 > ref1 + kQ8Step)) {
#pragma unroll
                    for (int sh = 4; sh < 32; sh <<= 1) {
                        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, sh));
                        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, sh));
                    }
                    m0 = fmaxf(m0, ref0);
                    m1 = fmaxf(m1, ref1);
                    const float c0 = ex2(ref0 - m0), c1 = ex2(ref1 - m1);
                    ref0 = m0;
                    ref1 = m1;
                    l0 *= c0;
                    l1 *= c1;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[j][0] *= c0;
                        o[j][1] *= c1;
                        o[j][2] *= c0;
                        o[j][3] *= c1;
                    }
                }
                const float s0 = ref0 - kQ8Top, s1 = ref1 - kQ8Top;
                const float p0 = ex2(x[0] - s0), p1 = ex2(x[1] - s1), p2 = ex2(x[2] - s0), p3 = ex2(x[3] - s1);
                l0 = fmaf(p2, rb, fmaf(p0, ra, l0));
                l1 = fmaf(p3, rb, fmaf(p1, ra, l1));
                const uint32_t ha = pack_h2(p0, p1), hb = pack_h2(p2, p3);
                const uint32_t ph0 = movmatrix(ha), ph1 = movmatrix(hb);
                uint32_t pl0 = 0u, pl1 = 0u;
                if constexpr (kLo) {
                    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&ha)), fb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
                    pl0 = movmatrix(pack_h2(p0 - fa.x, p1 - fa.y));
                    pl1 = movmatrix(pack_h2(p2 - fb.x, p3 - fb.y));
                }
                // O^T += V^T.P^T: product j has the dims 16 g + 2 j and 16 g + 2 j + 1 as its rows g and g + 8
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                    uint32_t wd[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) wd[e] = k4 == 0 ? vw[e].x : k4 == 1 ? vw[e].y : k4 == 2 ? vw[e].z : vw[e].w;
                    uint32_t b[2][4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {           // keys (2t, 2t+1), then (2t+8, 2t+9): codes of a dim side by side
                        q8_to_h2<kFmt>(__byte_perm(wd[2 * e], wd[2 * e + 1], 0x5140), b[e][0], b[e][1]);
                        q8_to_h2<kFmt>(__byte_perm(wd[2 * e], wd[2 * e + 1], 0x7362), b[e][2], b[e][3]);
                    }
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        mma_full(o[2 * k4 + d], b[0][2 * d], b[0][2 * d + 1], b[1][2 * d], b[1][2 * d + 1], ph0, ph1);
                        if constexpr (kLo) mma_full(o[2 * k4 + d], b[0][2 * d], b[0][2 * d + 1], b[1][2 * d], b[1][2 * d + 1], pl0, pl1);
                    }
                }
            }
            else if (lane == 0) {
                mbar_arrive(smem_u32(&s_empty[stage]));
            }
            stage += kSub;
            if (stage >= kStages) {
                stage -= kStages;
                parity ^= 1;
            }
        }
        it = it_end;

        // ---- the row's segment is done: the sums of the key lanes together, then the head's warps, then memory
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, sh);
            l1 += __shfl_xor_sync(0xffffffffu, l1, sh);
        }
        // every warp leaves its 32 sums a lane; each then adds up and writes some of them: piece un is four dims of a lane's head
        // 2 t + (un & 1), o[j][e] and o[j][2 + e] being the dims 16 g + 2 j and 16 g + 2 j + 1
        float* const all = merge + (size_t)w * kSub * 36 * 32 + lane;
        {
            float* p = all + (size_t)sub * 36 * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j) p[32 * j] = o[j >> 2][j & 3];
            p[32 * 32] = ref0;
            p[33 * 32] = ref1;
            p[34 * 32] = l0;
            p[35 * 32] = l1;
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");
#pragma unroll 1                                              // (unrolled, it waits longer for its instructions than it saves)
        for (int un = sub; un < 8; un += kSub) {
            const int e = un & 1, j = un & 6, hd = 2 * t + e;
            float M = -INFINITY, L = 0.f;
            float wt[kSub];
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                wt[u] = all[(size_t)u * 36 * 32 + 32 * (32 + e)];
                M = fmaxf(M, wt[u]);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < kSub; ++u) {
                const float* p = all + (size_t)u * 36 * 32;
                const float l = p[32 * (34 + e)], c = l != 0.f ? ex2(wt[u] - M) : 0.f;      // (a NaN stays one)
                L = fmaf(l, c, L);
                y = make_float4(fmaf(p[32 * (4 * j + e)], c, y.x), fmaf(p[32 * (4 * j + 2 + e)], c, y.y), fmaf(p[32 * (4 * j + 4 + e)], c, y.z),
                                fmaf(p[32 * (4 * j + 6 + e)], c, y.w));
            }
            if (hd >= G) continue;
            if (sg.whole) {
                const float inv = L > 0.f ? 1.f / L : 0.f;
                q8_store4(a.out, (int64_t)row * a.out_stride + (int64_t)(kvh * G + hd) * kHeadDim + 16 * g + 2 * j, a.io,
                          make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                float* p = a.part + ((size_t)((int)blockIdx.x + sg.row) * heads_per_row + (size_t)(w * G + hd)) * kSlotW;
                if (g == 0 && j == 0) *reinterpret_cast<float2*>(p) = make_float2(M, L);
                *reinterpret_cast<float4*>(p + 4 + 16 * g + 2 * j) = y;
            }
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");
    }
    dec_settle(&s_abort);
}

// Merge of the rows that several CTAs worked on: W warps per (row, head).  The first finds every contributor's weight; the
// contributors are dealt to the warps, eight at a time, a lane four dims; the warps' sums are added in order.
template <int W>
__global__ void __launch_bounds__(W == 16 ? 512 : 128) q8_decode_merge_kernel(Q8Launch a, int kvg, int grid_split) {
    constexpr int kWarps = W == 16 ? 16 : 4, kUnits = kWarps / W;
    __shared__ DecPlan s_plan;
    __shared__ float s_w[kUnits][kQ8MaxCtas];
    __shared__ float s_inv[kUnits];
    __shared__ float4 s_acc[W == 1 ? 1 : kWarps * 32];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, mine = warp / W, part = warp % W;
    const int G = a.n_heads / a.n_kv_heads, n_groups = a.n_kv_heads / kvg, heads_per_row = kvg * G;
    pdl_launch_dependents();
    dec_build_plan(a, s_plan, n_groups, false);           // (positions and row starts: written before the split, which waited)
    const DecLine ln = dec_line(a, s_plan, n_groups, grid_split);
    const int units = ln.total > 0 ? ln.rows * heads_per_row : 0;
    auto sync = [] {
        if constexpr (W == 1) __syncwarp();
        else __syncthreads();
    };
    // contributors of a unit: CTAs c0 .. c0 + n - 1 (n == 1: written by the split kernel)
    int r = 0, hr = 0, c0 = 0, n = 1;
    auto find = [&](int u) {
        n = 1;
        if (u >= units) return;
        r = u / heads_per_row;
        hr = u - r * heads_per_row;
        if (s_plan.prefix[r + 1] == s_plan.prefix[r]) return;
        c0 = ln.owner(s_plan.prefix[r]);
        n = ln.owner(s_plan.prefix[r + 1] - 1) - c0 + 1;
    };
    int u = (int)blockIdx.x * kUnits + mine;
    find(u);
    pdl_wait();
    for (; u < units; u += (int)gridDim.x * kUnits, find(u)) {
        if (n == 1) continue;
        const size_t step = (size_t)heads_per_row * kSlotW;
        const float* base = a.part + ((size_t)(c0 + r) * heads_per_row + hr) * kSlotW;
        constexpr int kBatch = W == 16 ? kQ8MaxCtas / W : 8;
        float4 x[kBatch];
        auto bring = [&](int i0) {
#pragma unroll
            for (int e = 0; e < kBatch; ++e)
                if (i0 + e * W < n) x[e] = __ldcg(reinterpret_cast<const float4*>(base + (size_t)(i0 + e * W) * step + 4 + 4 * lane));
        };
        bring(part);
        if (part == 0) {
            float2 ml[kQ8MaxCtas / 32];
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int e = 0; e < kQ8MaxCtas / 32; ++e) {
                ml[e] = make_float2(-INFINITY, 0.f);
                if (32 * e + lane < n) ml[e] = __ldcg(reinterpret_cast<const float2*>(base + (size_t)(32 * e + lane) * step));
            }
#pragma unroll
            for (int e = 0; e < kQ8MaxCtas / 32; ++e)
                if (ml[e].y != 0.f) M = fmaxf(M, ml[e].x);
#pragma unroll
            for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll
            for (int e = 0; e < kQ8MaxCtas / 32; ++e) {
                const float c = ml[e].y != 0.f ? ex2(ml[e].x - M) : 0.f;
                L += ml[e].y * c;
                if (32 * e + lane < n) s_w[mine][32 * e + lane] = c;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            if (lane == 0) s_inv[mine] = L > 0.f ? 1.f / L : 0.f;
        }
        sync();
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = part; i0 < n; i0 += kBatch * W) {
            if (i0 != part) bring(i0);
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (i0 + e * W >= n) break;
                const float c = s_w[mine][i0 + e * W];
                y = make_float4(fmaf(x[e].x, c, y.x), fmaf(x[e].y, c, y.y), fmaf(x[e].z, c, y.z), fmaf(x[e].w, c, y.w));
            }
        }
        if constexpr (W > 1) {
            s_acc[threadIdx.x] = y;
            sync();
            if (part == 0) {
#pragma unroll
                for (int v = 1; v < (n < W ? n : W); ++v) {
                    const float4 z = s_acc[32 * v + lane];
                    y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                }
            }
        }
        if (part == 0) {
            const float inv = s_inv[mine];
            const int s = r / n_groups, head = (r - s * n_groups) * heads_per_row + hr;
            q8_store4(a.out, (int64_t)s_plan.row[s] * a.out_stride + (int64_t)head * kHeadDim + 4 * lane, a.io,
                      make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
        }
        sync();
    }
}

template <int W>
cudaError_t merge_as(const Q8Launch& a, int kvg, int ctas, cudaStream_t s) {
    constexpr int kUnits = W == 1 ? 4 : 1;
    const int64_t units = ((int64_t)a.n_sessions * a.n_heads + kUnits - 1) / kUnits, cap = 4 * sm_count();
    return launch_kernel_pdl(q8_decode_merge_kernel<W>, dim3((unsigned)(units < cap ? units : cap)), dim3(W == 16 ? 512 : 128), 0, s, true, a, kvg, ctas);
}

int dec_group(int n_kv_heads) { return n_kv_heads % 4 == 0 ? 4 : (n_kv_heads % 2 == 0 ? 2 : 1); }

template <int KVG, int kFmt, bool kLo>
int launch_decode_as(const Q8Launch& a, const CUtensorMap& tmk, const CUtensorMap& tmv, int ctas, cudaStream_t s) {
    using Cfg = DecCfg<KVG>;
    NOVA_CUDA_TRY((q8_allow_smem<q8_decode_kernel<KVG, kFmt, kLo>>(Cfg::kSmem)));
    const cudaError_t e = launch_kernel_pdl(q8_decode_kernel<KVG, kFmt, kLo>, dim3((unsigned)ctas), dim3(Cfg::kThreads), (size_t)Cfg::kSmem, s, true, a, tmk, tmv);
    if (e != cudaSuccess) {
        set_cuda_error(e, "8-bit decode attention launch");
        return NOVA_ERR_CUDA;
    }
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

template <int KVG, int kFmt>
int launch_decode(const Q8Launch& a, const CUtensorMap& tmk, const CUtensorMap& tmv, int ctas, cudaStream_t s) {
    return a.io != NOVA_IO_BF16 && !a.one_part ? launch_decode_as<KVG, kFmt, true>(a, tmk, tmv, ctas, s) : launch_decode_as<KVG, kFmt, false>(a, tmk, tmv, ctas, s);
}

}  // namespace

bool q8_is_decode(int n_heads, int n_kv_heads, int max_tokens) { return max_tokens <= 1 && n_heads / n_kv_heads <= 8; }

size_t q8_work_bytes(int n_heads, int n_kv_heads, int n_sessions, int, int max_tokens) {
    if (!q8_is_decode(n_heads, n_kv_heads, max_tokens)) return q8_chunk_work_bytes(n_heads, n_kv_heads, max_tokens);
    const int kvg = dec_group(n_kv_heads), groups = n_kv_heads / kvg;
    const int64_t rows = (int64_t)n_sessions * groups;
    return (size_t)((rows < kDecRows ? rows : kDecRows) + kQ8MaxCtas) * (size_t)(kvg * (n_heads / n_kv_heads)) * kSlotW * sizeof(float);
}

int launch_q8_attn(const Q8Launch& call, cudaStream_t s) {
    if (call.n_tokens <= 0 || call.n_sessions <= 0) return NOVA_OK;
    Q8Launch a = call;
    a.keys_cap = (int)(a.table_stride > (kQ8MaxPos >> a.kv_shift) ? kQ8MaxPos : a.table_stride << a.kv_shift);
    if (q8_is_decode(a.n_heads, a.n_kv_heads, a.max_tokens)) {
        const int kvg = dec_group(a.n_kv_heads), groups = a.n_kv_heads / kvg;
        if (groups > kDecRows) return NOVA_ERR_TOO_LARGE;
        alignas(64) CUtensorMap tmk, tmv;
        const int64_t slot_rows = ((int64_t)(a.layer + 1) * a.nb) << a.kv_shift;
        const int box = a.kv_shift == 3 ? 8 : 16;
        int rc = attn_make_tmap(&tmk, a.pool_k, slot_rows, a.n_kv_heads, kvg, box, 1);
        if (rc == NOVA_OK) rc = attn_make_tmap(&tmv, a.pool_v, slot_rows, a.n_kv_heads, kvg, box, 1);
        if (rc != NOVA_OK) return rc;
        int ctas = sm_count();
        if (ctas > kQ8MaxCtas) ctas = kQ8MaxCtas;
        const int most = kDecRows / groups;                    // sessions of one launch (the row table's size)
        const int all = a.n_sessions;
        const size_t io_bytes = a.io == NOVA_IO_F32 ? 4 : 2;
        auto ahead = [&](const void* p, int64_t elems) -> const void* { return p ? static_cast<const unsigned char*>(p) + elems * (int64_t)io_bytes : nullptr; };
        for (int s0 = 0; s0 < all; s0 += most) {
            Q8Launch b = a;
            b.n_sessions = all - s0 < most ? all - s0 : most;
            b.n_past = a.n_past + s0;
            if (a.slice_ids) b.slice_ids = a.slice_ids + s0;
            else b.tables = a.tables + (int64_t)s0 * a.table_stride;
            if (a.tok_start) {
                b.tok_start = a.tok_start + s0;
            } else {                                                // one row per session
                b.q = ahead(a.q, s0 * a.q_stride);
                b.k = ahead(a.k, s0 * a.k_stride);
                b.v = ahead(a.v, s0 * a.v_stride);
                b.out = const_cast<void*>(ahead(a.out, s0 * a.out_stride));
                if (a.k_rot) b.k_rot = a.k_rot + (int64_t)s0 * a.n_kv_heads * kHeadDim;
            }
            rc = NOVA_ERR_UNSUPPORTED;
            if (a.fmt == NOVA_KV_I8) {
                if (kvg == 4) rc = launch_decode<4, NOVA_KV_I8>(b, tmk, tmv, ctas, s);
                else if (kvg == 2) rc = launch_decode<2, NOVA_KV_I8>(b, tmk, tmv, ctas, s);
                else rc = launch_decode<1, NOVA_KV_I8>(b, tmk, tmv, ctas, s);
            } else {
                if (kvg == 4) rc = launch_decode<4, NOVA_KV_E4M3>(b, tmk, tmv, ctas, s);
                else if (kvg == 2) rc = launch_decode<2, NOVA_KV_E4M3>(b, tmk, tmv, ctas, s);
                else rc = launch_decode<1, NOVA_KV_E4M3>(b, tmk, tmv, ctas, s);
            }
            if (rc != NOVA_OK) return rc;
            const int per_row = ctas / (b.n_sessions * groups);           // contributors of a row
            const cudaError_t e = per_row > 16 ? merge_as<16>(b, kvg, ctas, s) : per_row > 4 ? merge_as<4>(b, kvg, ctas, s) : merge_as<1>(b, kvg, ctas, s);
            if (e != cudaSuccess) {
                set_cuda_error(e, "8-bit decode merge launch");
                return NOVA_ERR_CUDA;
            }
            NOVA_LAUNCH_CHECK();
        }
        return NOVA_OK;
    }
    if (a.append) {
        const int rc = launch_q8_append(a, s);
        if (rc != NOVA_OK) return rc;
    }
    return launch_q8_chunk(a, s);
}

}  // namespace novab
