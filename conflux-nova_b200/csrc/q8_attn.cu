// q8_attn.cu — attention over the 8-bit paged cache: o = sum_j p_j v_j / sum_j p_j with p_j = exp(q.k_j / sqrt(128)), over the
// keys that a query sees (causal, or a sliding window of them), k_j and v_j = code * scale.
//
// One warp per (token, query head), a lane owns four dims; online softmax in fp32.
#include "q8_common.cuh"

namespace novab {
namespace {

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

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
    if (a.rope_cs) {
        float x[4] = {q.x, q.y, q.z, q.w}, y[4];
        const int i0 = a.neox ? 4 * (lane & 15) : 2 * lane;
        for (int e = 0; e < 4; ++e) {
            const float other = a.neox ? __shfl_xor_sync(0xffffffffu, x[e], 16) : x[e ^ 1];
            const int i = a.neox ? i0 + e : i0 + (e >> 1);
            const float c = a.rope_cs[pos * 64 + i], sn = a.rope_sn[pos * 64 + i];
            const bool lower = a.neox ? lane < 16 : !(e & 1);
            y[e] = lower ? __fmaf_rn(x[e], c, -__fmul_rn(other, sn)) : __fmaf_rn(other, sn, __fmul_rn(x[e], c));
        }
        q = make_float4(y[0], y[1], y[2], y[3]);
    }
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

}  // namespace

size_t q8_work_bytes(int, int, int, int, int) { return 0; }

int launch_q8_attn(const Q8Launch& a, size_t, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    const int64_t blocks = ((int64_t)a.n_tokens * a.n_heads + 3) / 4;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    if (a.fmt == NOVA_KV_I8) q8_attn_kernel<NOVA_KV_I8><<<(unsigned)blocks, 128, 0, s>>>(a);
    else q8_attn_kernel<NOVA_KV_E4M3><<<(unsigned)blocks, 128, 0, s>>>(a);
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

}  // namespace novab
