// q8_attn.cu — attention over the 8-bit paged cache: o = sum_j p_j v_j / sum_j p_j with p_j = exp(q.k_j / sqrt(128)), over the
// keys that a query sees (causal, or a sliding window of them), k_j and v_j = code * scale.
//
// This file: single new tokens (decode).  What bounds it is HBM: 264 bytes per key and kv head (two rows of codes, two
// scales), against 4 * 128 * G flops.
//
//   * One persistent CTA per SM; the 16-key tiles of all (session, kv group) rows form one line that is dealt out evenly
//     (attn_plan.cuh); rows that several CTAs worked on are merged by the kernel behind it.
//   * A producer warp brings the tiles in with TMA: boxes [128 B][16 slots][kv group] of codes, 128-byte swizzle (a row of codes
//     is one swizzle line), and the tile's scales with plain bulk copies.
//   * Eight consumer warps: 8 / KVG of them per kv head, each with its own running maximum, sums and accumulators over every
//     (8 / KVG)-th tile; merged once per row.  Codes become fp16 in registers (exactly: both formats fit fp16's mantissa)
//     and go to mma.sync m16n8k16.  A lane reads 32 consecutive codes of a key: the contraction index of S = Q.K^T may be permuted
//     freely as long as q's fragments follow, so no transposition is needed; for P.V the columns are permuted the same
//     way (column n of product j is dim 16 n + j) and pairs of keys are interleaved with byte permutes.
//   * The at most 8 query heads of a kv head fill half of the 16 rows.  The other half holds the low parts: q = hi + lo and
//     p = hi + lo in fp16, both halves in one instruction, so scores and outputs keep fp32-level accuracy at no cost.
//   * The scale of K multiplies the finished score.  The scale of V goes into the exponent: w_j = 2^(x_j + log2 sv_j - m), so
//     the weights that multiply the codes never leave fp16's range whatever the scales are; the softmax sum adds w_j / sv_j.
#include "attn_plan.cuh"
#include "mma_common.cuh"
#include "q8_common.cuh"

namespace novab {
namespace {

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two codes (the low 16 bits of lo16: first code in the low byte) ... four codes of a word -> two pairs of fp16, exactly.
template <int kFmt> __device__ __forceinline__ void q8_to_h2(uint32_t w, uint32_t& h0, uint32_t& h1) {
    if constexpr (kFmt == NOVA_KV_I8) {
        // 0x6400 | (code + 128) is the fp16 number 1024 + 128 + code
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), k), y = __hsub2(*reinterpret_cast<const __half2*>(&b), k);
        h0 = *reinterpret_cast<const uint32_t*>(&x);
        h1 = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }" : "=r"(h0), "=r"(h1) : "r"(w));
    }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float2 lds_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

constexpr int kSetupTiles = 2;       // work-split weight of starting a row inside a CTA, in tiles
constexpr int kMinTiles = 4;         // a CTA gets at least that many tiles (fewer partial rows to merge for short contexts)

template <int KVG>
struct DecCfg {
    static constexpr int kSub = 8 / KVG;                    // consumer warps per kv head
    static constexpr int kStages = 32 / KVG;                // 128 KiB of tiles in flight
    static constexpr int kHalf = KVG * 2048;                // K (or V) codes of a tile
    static constexpr int kTile = 2 * kHalf;
    static constexpr int kScales = KVG * 128;               // K scales | V scales
    static constexpr int kMergeFloats = KVG * (kSub - 1) * 34 * 32;
    static constexpr int kSmem = kStages * (kTile + kScales) + kMergeFloats * 4 + 1024;
    static constexpr int kThreads = 288;
};

// Keys, first tile and tile count of every (session, group) row; a row without a new token has no tiles.
struct DecPlan {
    int prefix[kMaxRowsSmem + 1];
    int keys[kMaxRowsSmem];
    int row[kMaxRowsSmem];
    int slice[kMaxRowsSmem];
};

__device__ __forceinline__ int dec_first_tile(const Q8Launch& a, int keys) { return a.window > 0 && keys > a.window ? (keys - a.window) >> 4 : 0; }

__device__ inline void dec_build_plan(const Q8Launch& a, DecPlan& p, int n_groups, bool flag) {
    if (threadIdx.x < 32) {
        const int lane = (int)threadIdx.x, rows = a.n_sessions * n_groups;
        int carry = 0;
        if (lane == 0) p.prefix[0] = 0;
        for (int base = 0; base < rows; base += 32) {
            const int r = base + lane;
            int v = 0;
            if (r < rows) {
                const int s = r / n_groups;
                int first, count;
                q8_rows(a, s, first, count);
                const int pos = __ldg(a.n_past + s);
                int keys = 0;
                if (count > 0) {
                    if (pos < 0 || pos == 0x7fffffff || (a.rope_cs && pos >= a.rope_rows)) {
                        if (flag) q8_flag(a, NOVA_ERR_INVALID);
                    } else {
                        keys = pos + 1;
                    }
                }
                if (r - s * n_groups == 0) {
                    p.keys[s] = keys;
                    p.row[s] = first;
                    p.slice[s] = a.slice_ids ? __ldg(a.slice_ids + s) : s;
                }
                v = keys > 0 ? ((keys + 15) >> 4) - dec_first_tile(a, keys) + kSetupTiles : 0;
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += t;
            }
            if (r < rows) p.prefix[r + 1] = carry + v;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}

__device__ __forceinline__ PlanView dec_view(const Q8Launch& a, const DecPlan& p, int n_groups, int grid) {
    PlanView pv;
    pv.prefix = p.prefix;
    pv.rows_per_layer = a.n_sessions * n_groups;
    pv.n_groups = n_groups;
    pv.pages_per_layer = p.prefix[pv.rows_per_layer];
    pv.pages_total = pv.pages_per_layer;
    const int64_t most = (pv.pages_total + kMinTiles - 1) / kMinTiles;
    pv.n_ctas = most < grid ? (int)most : grid;
    plan_finish(pv);
    return pv;
}

template <int KVG, int kFmt>
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
    float* const merge = reinterpret_cast<float*>(smem_raw + (scale0 - smem_u32(smem_raw)) + kStages * Cfg::kScales);
    // a page of 8 tokens is half a tile: two boxes of 8 slots, [half][kv head][8]; otherwise [kv head][16]
    const bool p8 = a.kv_shift == 3;
    const uint32_t head_step = p8 ? 1024u : 2048u, half_step = p8 ? KVG * 1024u : 1024u;
    const uint32_t sc_head = p8 ? 32u : 64u, sc_half = p8 ? KVG * 32u : 32u;

    if (threadIdx.x == 256) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
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
    const PlanView pv = dec_view(a, s_plan, n_groups, (int)gridDim.x);
    if (pv.pages_total == 0 || (int)blockIdx.x >= pv.n_ctas) return;
    const int64_t lo = plan_cta_begin(pv, (int)blockIdx.x), hi = plan_cta_begin(pv, (int)blockIdx.x + 1);

    // ------------------------------------------------------------------------------------------------ producer
    if (warp == 8) {
        const unsigned long long policy = l2_policy_evict_first();
        // what this lane copies of every tile: K or V codes (one box, or one per page of 8), K or V scales (one run of the kv
        // group per page of 8 or 16, one run per head in longer pages)
        const int n_box = p8 ? 2 : 1, n_sc = p8 ? 2 : (a.kv_shift == 4 ? 1 : KVG), jobs = 2 * (n_box + n_sc);
        const bool is_box = lane < 2 * n_box;
        const int j = is_box ? lane : lane - 2 * n_box;
        const bool is_v = j >= (is_box ? n_box : n_sc);
        const int part = is_v ? j - (is_box ? n_box : n_sc) : j;           // page of the tile, or head
        const uint32_t sc_bytes = (uint32_t)(p8 ? KVG * 32 : (a.kv_shift == 4 ? KVG * 64 : 64));
        const uint32_t my_off = is_box ? (uint32_t)(is_v ? Cfg::kHalf : 0) + (p8 ? part * half_step : 0u)
                                       : (uint32_t)(is_v ? KVG * 64 : 0) + part * sc_bytes;
        const float* const my_scale = is_v ? a.scale_v : a.scale_k;
        const int tpp = a.kv_shift > 4 ? a.kv_shift - 4 : 0;               // log2(tiles per page)
        uint32_t it = 0;
        for (int64_t pos = lo; pos < hi;) {
            const Segment sg = plan_segment(pv, pos, hi, kSetupTiles);
            pos += sg.span;
            const int keys = s_plan.keys[sg.session];
            const int t0 = dec_first_tile(a, keys) + sg.page_first, low = a.window > 0 && keys > a.window ? keys - a.window : 0;
            const int32_t* table = a.tables + (int64_t)s_plan.slice[sg.session] * a.table_stride;
            auto entry = [&](int64_t page, int first_key) -> int {        // block-table entry of a page that starts at first_key
                if (first_key >= keys) return -2;                           // behind the last key: nothing to bring
                if (page >= a.table_stride) return -1;
                const int e = __ldg(table + page);
                return e >= 0 && e < a.nb ? e : -1;
            };
            auto fetch = [&](int t, int& e0, int& e1) {
                e0 = e1 = -2;
                if (t < t0 + sg.page_count) {
                    if (p8) {
                        e0 = entry(2 * (int64_t)t, 16 * t);
                        e1 = entry(2 * (int64_t)t + 1, 16 * t + 8);
                    } else {
                        e0 = entry(t >> tpp, 16 * t);
                    }
                }
            };
            int n0, n1;
            fetch(t0 + lane, n0, n1);
            for (int b = 0; b < sg.page_count; b += 32) {
                const int c0 = n0, c1 = n1;
                fetch(t0 + b + 32 + lane, n0, n1);
                const int n = sg.page_count - b < 32 ? sg.page_count - b : 32;
                for (int i = 0; i < n; ++i, ++it) {
                    const int e0 = __shfl_sync(0xffffffffu, c0, i), e1 = __shfl_sync(0xffffffffu, c1, i);
                    const int t = t0 + b + i, stage = (int)(it % kStages);
                    const uint32_t round = it / kStages;
                    if (round > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_empty[stage]), (round - 1) & 1, &s_abort))) {
                        if (lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);
                        return;
                    }
                    const uint32_t bar = smem_u32(&s_full[stage]);
                    if (lane == 0) {
                        if (e0 == -1 || e1 == -1) q8_flag(a, NOVA_ERR_BAD_TABLE);
                        uint32_t mask = p8 ? (e0 >= 0 ? 0xffu : 0u) | (e1 >= 0 ? 0xff00u : 0u) : (e0 >= 0 ? 0xffffu : 0u);
                        if (keys - 16 * t < 16) mask &= (1u << (keys - 16 * t)) - 1u;
                        if (low > 16 * t) mask &= ~((1u << (low - 16 * t < 16 ? low - 16 * t : 16)) - 1u);
                        s_mask[stage] = mask;
                        s_phys[stage] = p8 && e1 >= 0 ? e1 : e0;
                        const uint32_t bytes = (uint32_t)(p8 ? ((e0 >= 0) + (e1 >= 0)) * (Cfg::kTile + Cfg::kScales) / 2 : (e0 >= 0 ? Cfg::kTile + Cfg::kScales : 0));
                        if (bytes) mbar_expect_tx(bar, bytes);
                        else mbar_arrive(bar);
                    }
                    __syncwarp();
                    if (lane < jobs) {
                        const int e = p8 && part == 1 ? e1 : e0;
                        if (e >= 0) {
                            const int64_t page = (int64_t)a.layer * a.nb + e;
                            const int slot = p8 ? 0 : (t << 4) & ((1 << a.kv_shift) - 1);
                            if (is_box) {
                                tma_load_3d_hint(tile0 + (uint32_t)stage * Cfg::kTile + my_off, is_v ? &tmv : &tmk, 0, (int)((page << a.kv_shift) + slot),
                                                 sg.group * KVG, bar, policy);
                            } else {
                                const int h = sg.group * KVG + (a.kv_shift > 4 ? part : 0);
                                bulk_load(scale0 + (uint32_t)stage * Cfg::kScales + my_off, my_scale + ((page * a.n_kv_heads + h) << a.kv_shift) + slot, sc_bytes, bar);
                            }
                        }
                    }
                }
            }
        }
        return;
    }

    // ------------------------------------------------------------------------------------------------ consumers
    const int w = warp % KVG, sub = warp / KVG;       // kv head of the group, which of its warps
    const int g = lane >> 2, t = lane & 3;
    constexpr float kToLog2 = kAttnScale * kLog2e * 8.f;      // q goes in divided by 8: rotated fp16 values stay inside fp16
    uint32_t it = 0;
    for (int64_t pos = lo; pos < hi;) {
        const Segment sg = plan_segment(pv, pos, hi, kSetupTiles);
        pos += sg.span;
        const int s = sg.session, kvh = sg.group * KVG + w;
        const int keys = s_plan.keys[s], row = s_plan.row[s], t0 = dec_first_tile(a, keys) + sg.page_first;
        const int head = kvh * G + (g < G ? g : 0);

        // q fragments of head g: this lane's dims are 32 t .. 32 t + 31 (four per contraction step), rows 8-15 hold the low parts
        uint32_t qh[8][2], ql[8][2];
        {
            const int64_t qe = (int64_t)row * a.q_stride + (int64_t)head * kHeadDim;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                float4 x = q8_load4(a.q, qe + 32 * t + 4 * ks, a.io);
                if (a.rope_cs) {
                    const int64_t cpos = (int64_t)(keys - 1) * 64;
                    if (a.neox) {
                        const float4 y = q8_load4(a.q, qe + ((32 * t) ^ 64) + 4 * ks, a.io);
                        const float4 c = *reinterpret_cast<const float4*>(a.rope_cs + cpos + ((32 * t) & 63) + 4 * ks);
                        const float4 n = *reinterpret_cast<const float4*>(a.rope_sn + cpos + ((32 * t) & 63) + 4 * ks);
                        if (t < 2) x = make_float4(__fmaf_rn(x.x, c.x, -__fmul_rn(y.x, n.x)), __fmaf_rn(x.y, c.y, -__fmul_rn(y.y, n.y)),
                                                   __fmaf_rn(x.z, c.z, -__fmul_rn(y.z, n.z)), __fmaf_rn(x.w, c.w, -__fmul_rn(y.w, n.w)));
                        else x = make_float4(__fmaf_rn(y.x, n.x, __fmul_rn(x.x, c.x)), __fmaf_rn(y.y, n.y, __fmul_rn(x.y, c.y)),
                                             __fmaf_rn(y.z, n.z, __fmul_rn(x.z, c.z)), __fmaf_rn(y.w, n.w, __fmul_rn(x.w, c.w)));
                    } else {
                        const float2 c = *reinterpret_cast<const float2*>(a.rope_cs + cpos + 16 * t + 2 * ks);
                        const float2 n = *reinterpret_cast<const float2*>(a.rope_sn + cpos + 16 * t + 2 * ks);
                        x = make_float4(__fmaf_rn(x.x, c.x, -__fmul_rn(x.y, n.x)), __fmaf_rn(x.x, n.x, __fmul_rn(x.y, c.x)),
                                        __fmaf_rn(x.z, c.y, -__fmul_rn(x.w, n.y)), __fmaf_rn(x.z, n.y, __fmul_rn(x.w, c.y)));
                    }
                }
                const float f[4] = {x.x * 0.125f, x.y * 0.125f, x.z * 0.125f, x.w * 0.125f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
                    const float2 b = __half22float2(h);
                    qh[ks][e] = g < G ? *reinterpret_cast<const uint32_t*>(&h) : 0u;
                    ql[ks][e] = g < G ? pack_h2(f[2 * e] - b.x, f[2 * e + 1] - b.y) : 0u;
                }
            }
        }
        float m = -INFINITY, l = 0.f;
        float o[16][4];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

        const uint32_t it_end = it + (uint32_t)sg.page_count;
        for (uint32_t i = it + (((uint32_t)sub + kSub - it % kSub) % kSub); i < it_end; i += kSub) {
            const int stage = (int)(i % kStages);
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[stage]), (i / kStages) & 1, &s_abort))) {
                if (lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);      // the result is void; the warp still meets its siblings below
                break;
            }
            const uint32_t mask = s_mask[stage];
            const uint32_t sk = tile0 + (uint32_t)stage * Cfg::kTile + w * head_step, sv = sk + Cfg::kHalf;
            const uint32_t ck = scale0 + (uint32_t)stage * Cfg::kScales + w * sc_head, cv = ck + KVG * 64;
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
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"((i2 ? cv : ck) + (slot >> 3) * sc_half + (slot & 7) * 4u), "f"(scale) : "memory");
                    }
                }
                __syncwarp();
            }
            if (mask) {
                // S = Q.K^T: lane (g, t) holds codes 32 t .. of keys g and g + 8 (two swizzled 16-byte pieces each)
                float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint4 kw[2];
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) kw[nt] = lds128(sk + nt * half_step + g * 128u + (((2 * t + half) ^ g) << 4));
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const int ks = 4 * half + k4;
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            uint32_t b0, b1;
                            q8_to_h2<kFmt>(k4 == 0 ? kw[nt].x : k4 == 1 ? kw[nt].y : k4 == 2 ? kw[nt].z : kw[nt].w, b0, b1);
                            mma_full(c[nt], qh[ks][0], ql[ks][0], qh[ks][1], ql[ks][1], b0, b1);
                        }
                    }
                }
                uint4 vw[4];       // codes 16 g .. 16 g + 15 of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int e = 0; e < 4; ++e) vw[e] = lds128(sv + (e >> 1) * half_step + (2 * t + (e & 1)) * 128u + ((g ^ (2 * t + (e & 1))) << 4));
                float x[4], r[4];
                {
                    const float2 k0 = lds_f2(ck + 8 * t), k1 = lds_f2(ck + sc_half + 8 * t), v0 = lds_f2(cv + 8 * t), v1 = lds_f2(cv + sc_half + 8 * t);
                    const float fk[4] = {k0.x, k0.y, k1.x, k1.y}, fv[4] = {v0.x, v0.y, v1.x, v1.y};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float sv_e = fmaxf(fv[e], kQ8MinScale);
                        r[e] = rcp(sv_e);
                        x[e] = fmaf(c[e >> 1][e & 1] + c[e >> 1][2 + (e & 1)], fk[e] * kToLog2, lg2(sv_e));
                    }
                }
                if (mask != 0xffffu) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((mask >> (2 * t + (e & 1) + 8 * (e >> 1))) & 1)) {      // what is masked may hold anything
                            x[e] = -INFINITY;
                            r[e] = 0.f;
                            vw[e] = make_uint4(0u, 0u, 0u, 0u);
                        }
                }
                float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m, mx);
                if (__any_sync(0xffffffffu, mn != m)) {
                    const float corr = ex2(m - mn);
                    l *= corr;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        o[j][0] *= corr;
                        o[j][1] *= corr;
                        o[j][2] *= corr;
                        o[j][3] *= corr;
                    }
                    m = mn;
                }
                // The largest weight is 2^14, not 1: a weight of fp16 then keeps its 11 bits down to 2^-28 of the largest (2^14
                // cancels between the outputs and l).
                const float ref = m - 14.f;
                uint32_t ph[2], pl[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float p0 = ex2(x[2 * e] - ref), p1 = ex2(x[2 * e + 1] - ref);
                    l = fmaf(p0, r[2 * e], l);
                    l = fmaf(p1, r[2 * e + 1], l);
                    const __half2 h = __floats2half2_rn(p0, p1);
                    const float2 b = __half22float2(h);
                    ph[e] = *reinterpret_cast<const uint32_t*>(&h);
                    pl[e] = pack_h2(p0 - b.x, p1 - b.y);
                }
                // O += P.V: product j has the dims 16 n + j, n = 0..7, as its columns
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
                    for (int d = 0; d < 4; ++d) mma_full(o[4 * k4 + d], ph[0], pl[0], ph[1], pl[1], b[0][d], b[1][d]);
                }
            }
            if (patched) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
        }
        it = it_end;

        // ---- the row's segment is done: high and low parts together, then the head's warps, then memory
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        float acc[32];             // dims 32 t + i of head g
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            acc[j] = o[j][0] + o[j][2];
            acc[16 + j] = o[j][1] + o[j][3];
        }
        if constexpr (kSub > 1) {
            float* mine = merge + (size_t)(w * (kSub - 1)) * 34 * 32 + lane;
            if (sub > 0) {
                float* p = mine + (size_t)(sub - 1) * 34 * 32;
#pragma unroll
                for (int j = 0; j < 32; ++j) p[32 * j] = acc[j];
                p[32 * 32] = m;
                p[33 * 32] = l;
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");
            if (sub == 0) {
#pragma unroll 1
                for (int u = 0; u < kSub - 1; ++u) {
                    const float* p = mine + (size_t)u * 34 * 32;
                    const float mu = p[32 * 32], lu = p[33 * 32];
                    const float mn = fmaxf(m, mu);
                    const float c0 = m == -INFINITY ? 0.f : ex2(m - mn), c1 = mu == -INFINITY ? 0.f : ex2(mu - mn);
                    l = l * c0 + lu * c1;
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[j] = acc[j] * c0 + p[32 * j] * c1;
                    m = mn;
                }
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + w), "r"(32 * kSub) : "memory");
            if (sub > 0) continue;
        }
        if (g >= G) continue;
        if (sg.c_last == sg.c_first) {
            const float inv = l > 0.f ? 1.f / l : 0.f;
            const int64_t oe = (int64_t)row * a.out_stride + (int64_t)head * kHeadDim + 32 * t;
#pragma unroll
            for (int j = 0; j < 32; j += 4) q8_store4(a.out, oe + j, a.io, make_float4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv));
        } else {
            float* p = a.part + ((size_t)((int64_t)blockIdx.x + sg.row_id) * heads_per_row + (size_t)(w * G + g)) * kSlotW;
            if (t == 0) *reinterpret_cast<float2*>(p) = make_float2(m, l);
#pragma unroll
            for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(p + 4 + 32 * t + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        }
    }
}

// Merge of the rows that several CTAs worked on.  One CTA of four warps per (row, head); the warps take the contributors in
// turn, four at a time, a lane four dims; the warps' sums meet in shared memory, always in the same order.
__global__ void __launch_bounds__(128) q8_decode_merge_kernel(Q8Launch a, int kvg, int grid_split) {
    __shared__ DecPlan s_plan;
    __shared__ float s_ml[8];
    __shared__ float4 s_acc[128];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const int G = a.n_heads / a.n_kv_heads, n_groups = a.n_kv_heads / kvg, heads_per_row = kvg * G;
    pdl_launch_dependents();
    dec_build_plan(a, s_plan, n_groups, false);           // (positions and row starts: written before the split, which waited)
    const PlanView pv = dec_view(a, s_plan, n_groups, grid_split);
    const int units = pv.pages_total > 0 ? pv.rows_per_layer * heads_per_row : 0;
    pdl_wait();
    for (int u = (int)blockIdx.x; u < units; u += (int)gridDim.x) {
        const int r = u / heads_per_row, hr = u - r * heads_per_row;
        if (s_plan.prefix[r + 1] == s_plan.prefix[r]) continue;
        const int c0 = plan_owner(pv, s_plan.prefix[r]), n = plan_owner(pv, s_plan.prefix[r + 1] - 1) - c0 + 1;
        if (n == 1) continue;                              // written by the split kernel
        const size_t step = (size_t)heads_per_row * kSlotW;
        const float* base = a.part + ((size_t)(c0 + r) * heads_per_row + hr) * kSlotW;
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 4 * warp; i < n; i += 16) {
            float2 ml[4];
            float4 x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float* p = base + (size_t)(i + e < n ? i + e : i) * step;
                ml[e] = __ldcg(reinterpret_cast<const float2*>(p));
                x[e] = __ldcg(reinterpret_cast<const float4*>(p + 4 + 4 * lane));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e >= n || !(ml[e].y > 0.f)) continue;
                const float mn = fmaxf(M, ml[e].x), cm = M == -INFINITY ? 0.f : ex2(M - mn), cx = ex2(ml[e].x - mn);
                M = mn;
                L = L * cm + ml[e].y * cx;
                acc = make_float4(acc.x * cm + x[e].x * cx, acc.y * cm + x[e].y * cx, acc.z * cm + x[e].z * cx, acc.w * cm + x[e].w * cx);
            }
        }
        if (lane == 0) {
            s_ml[2 * warp] = M;
            s_ml[2 * warp + 1] = L;
        }
        s_acc[threadIdx.x] = acc;
        __syncthreads();
        if (warp == 0) {
            float Mx = -INFINITY, Lx = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int v = 0; v < 4; ++v) Mx = fmaxf(Mx, s_ml[2 * v]);
            for (int v = 0; v < 4; ++v) {
                if (s_ml[2 * v] == -INFINITY) continue;
                const float cw = ex2(s_ml[2 * v] - Mx);
                const float4 z = s_acc[32 * v + lane];
                Lx += s_ml[2 * v + 1] * cw;
                y = make_float4(y.x + z.x * cw, y.y + z.y * cw, y.z + z.z * cw, y.w + z.w * cw);
            }
            const float inv = Lx > 0.f ? 1.f / Lx : 0.f;
            const int s = r / n_groups, head = (r - s * n_groups) * heads_per_row + hr;
            q8_store4(a.out, (int64_t)s_plan.row[s] * a.out_stride + (int64_t)head * kHeadDim + 4 * lane, a.io,
                      make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
        }
        __syncthreads();
    }
}

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Several new tokens per session, or more than 8 query heads per kv head: one warp per (token, query head), a lane owns four
// dims; online softmax in fp32.
template <int kFmt>
__global__ void __launch_bounds__(128) q8_attn_kernel(Q8Launch a) {
    const int lane = (int)threadIdx.x & 31;
    const int64_t job = (int64_t)blockIdx.x * 4 + ((int)threadIdx.x >> 5);
    if (job >= (int64_t)a.n_tokens * a.n_heads) return;
    const int r = (int)(job / a.n_heads), head = (int)(job - (int64_t)r * a.n_heads);
    int t;
    const int s = q8_session_of(a, r, t);
    if (s < 0) return;
    const int64_t pos = (int64_t)__ldg(a.n_past + s) + t;
    if (pos < 0 || (a.rope_cs && pos >= a.rope_rows)) {
        if (lane == 0) q8_flag(a, NOVA_ERR_INVALID);
        return;
    }
    const int h = head / (a.n_heads / a.n_kv_heads);
    float4 q = q8_load4(a.q, (int64_t)r * a.q_stride + head * kHeadDim + 4 * lane, a.io);
    if (a.rope_cs) q = q8_rotate(q, pos, lane, a);
    const int64_t first = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const int32_t* table = q8_table(a, s);
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t j = first; j <= pos; ++j) {
        const int64_t lb = j >> a.kv_shift;
        const int phys = lb < a.table_stride ? __ldg(table + lb) : -1;
        if (phys < 0 || phys >= a.nb) {
            if (lane == 0) q8_flag(a, NOVA_ERR_BAD_TABLE);
            continue;
        }
        const int64_t page = (int64_t)a.layer * a.nb + phys;
        const int slot = (int)(j & ((1 << a.kv_shift) - 1));
        const int64_t row = (((page << a.kv_shift) + slot) * a.n_kv_heads + h) * kHeadDim + 4 * lane;
        const int64_t sc = ((page * a.n_kv_heads + h) << a.kv_shift) + slot;
        const float4 k = q8_decode4<kFmt>(*reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(a.pool_k) + row));
        const float4 v = q8_decode4<kFmt>(*reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(a.pool_v) + row));
        const float x = warp_total(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * (a.scale_k[sc] * kAttnScale);
        const float mn = fmaxf(m, x);
        const float corr = expf(m - mn), p = expf(x - mn), pv = p * a.scale_v[sc];
        m = mn;
        l = fmaf(l, corr, p);
        acc.x = fmaf(acc.x, corr, pv * v.x);
        acc.y = fmaf(acc.y, corr, pv * v.y);
        acc.z = fmaf(acc.z, corr, pv * v.z);
        acc.w = fmaf(acc.w, corr, pv * v.w);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    q8_store4(a.out, (int64_t)r * a.out_stride + head * kHeadDim + 4 * lane, a.io, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

int dec_group(int n_kv_heads) { return n_kv_heads % 4 == 0 ? 4 : (n_kv_heads % 2 == 0 ? 2 : 1); }
bool is_decode(int n_heads, int n_kv_heads, int max_tokens) { return max_tokens <= 1 && n_heads / n_kv_heads <= 8; }

template <int KVG, int kFmt>
int launch_decode(const Q8Launch& a, const CUtensorMap& tmk, const CUtensorMap& tmv, int ctas, cudaStream_t s) {
    using Cfg = DecCfg<KVG>;
    NOVA_CUDA_TRY((cudaFuncSetAttribute(q8_decode_kernel<KVG, kFmt>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem)));
    const cudaError_t e = launch_kernel_pdl(q8_decode_kernel<KVG, kFmt>, dim3((unsigned)ctas), dim3(Cfg::kThreads), (size_t)Cfg::kSmem, s, true, a, tmk, tmv);
    if (e != cudaSuccess) {
        set_cuda_error(e, "8-bit decode attention launch");
        return NOVA_ERR_CUDA;
    }
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

}  // namespace

size_t q8_work_bytes(int n_heads, int n_kv_heads, int n_sessions, int, int max_tokens) {
    if (!is_decode(n_heads, n_kv_heads, max_tokens)) return 0;
    const int kvg = dec_group(n_kv_heads), groups = n_kv_heads / kvg;
    const int64_t rows = (int64_t)n_sessions * groups;
    return (size_t)((rows < kMaxRowsSmem ? rows : kMaxRowsSmem) + kMaxSms) * (size_t)(kvg * (n_heads / n_kv_heads)) * kSlotW * sizeof(float);
}

int launch_q8_attn(const Q8Launch& a_in, size_t, cudaStream_t s) {
    Q8Launch a = a_in;
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    if (is_decode(a.n_heads, a.n_kv_heads, a.max_tokens)) {
        const int kvg = dec_group(a.n_kv_heads), groups = a.n_kv_heads / kvg;
        if (groups > kMaxRowsSmem) return NOVA_ERR_TOO_LARGE;
        alignas(64) CUtensorMap tmk, tmv;
        const int64_t slot_rows = ((int64_t)(a.layer + 1) * a.nb) << a.kv_shift;
        const int box = a.kv_shift == 3 ? 8 : 16;
        int rc = attn_make_tmap(&tmk, a.pool_k, slot_rows, a.n_kv_heads, kvg, box, 1);
        if (rc == NOVA_OK) rc = attn_make_tmap(&tmv, a.pool_v, slot_rows, a.n_kv_heads, kvg, box, 1);
        if (rc != NOVA_OK) return rc;
        int ctas = sm_count();
        if (ctas > kMaxSms) ctas = kMaxSms;
        const int most = kMaxRowsSmem / groups;                    // sessions of one launch (the row table's size)
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
            const int units = b.n_sessions * a.n_heads;
            const int cap = 4 * sm_count();
            const cudaError_t e = launch_kernel_pdl(q8_decode_merge_kernel, dim3((unsigned)(units < cap ? units : cap)), dim3(128), 0, s, true, b, kvg, ctas);
            if (e != cudaSuccess) {
                set_cuda_error(e, "8-bit decode merge launch");
                return NOVA_ERR_CUDA;
            }
            NOVA_LAUNCH_CHECK();
        }
        return NOVA_OK;
    }
    const int64_t blocks = ((int64_t)a.n_tokens * a.n_heads + 3) / 4;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    if (a.append) {
        const int rc = launch_q8_append(a, s);
        if (rc != NOVA_OK) return rc;
    }
    if (a.fmt == NOVA_KV_I8) q8_attn_kernel<NOVA_KV_I8><<<(unsigned)blocks, 128, 0, s>>>(a);
    else q8_attn_kernel<NOVA_KV_E4M3><<<(unsigned)blocks, 128, 0, s>>>(a);
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

}  // namespace novab
