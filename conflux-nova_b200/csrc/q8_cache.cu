// q8_cache.cu — writing the 8-bit paged cache and reading it back, and the C entry points of its operators.
//
// Writing: a row r (one token of one kv head; K rotated first where rotary tables are given, in the fused form of
// rope_append.cu) becomes  amax = max(max|r|, 2^-60),  scale = amax / Q,  code = rn(r * (Q / amax)),  Q = 127 (int8) or
// 448 (e4m3).  The three fp32 operations are rounded once each, so the codes are the same wherever the formula is followed.
// Reading: value = code * scale.
#include <cstring>
#include <type_traits>

#include "q8_common.cuh"

namespace novab {
namespace {

// A CTA takes kJobs consecutive (token, row) jobs - a token's rows are its K heads, its V heads and, where q is rotated in place
// too, its query heads - a warp eight of them, 16 lanes a row, 8 values a lane.  What the rows hold is asked for before it is
// known where they go (session, position, page: a chain of dependent loads, one thread per token), so that one wait covers
// both.  Bound by HBM: 2 * 128 * (io bytes) read and 2 * 132 written per token and kv head.
constexpr int kJobs = 64;
struct Place {
    int64_t page;      // page of the pools (layer included), or -1
    int64_t pos;       // position, or -1: nobody's row
    int slot;
};

__device__ __forceinline__ void q8_places(const Q8Launch& a, Place* places, int64_t job0, int units) {
    const int tok0 = (int)(job0 / units);
    const int64_t last = (job0 + kJobs - 1) / units;
    const int tok1 = last < a.n_tokens - 1 ? (int)last : a.n_tokens - 1;
    for (int i = (int)threadIdx.x; i <= tok1 - tok0; i += (int)blockDim.x) {
        Place p;
        p.page = p.pos = -1;
        p.slot = 0;
        int t;
        const int s = q8_session_of(a, tok0 + i, t);
        if (s >= 0) {
            const int64_t pos = (int64_t)__ldg(a.n_past + s) + t;
            if (pos < 0) {
                q8_flag(a, NOVA_ERR_INVALID);
            } else {
                p.pos = pos;
                const int64_t lb = pos >> a.kv_shift;
                const int phys = lb < a.table_stride ? __ldg(q8_table(a, s) + lb) : -1;
                if (phys >= 0 && phys < a.nb) p.page = (int64_t)a.layer * a.nb + phys;
                else q8_flag(a, NOVA_ERR_BAD_TABLE);
                p.slot = (int)(pos & ((1 << a.kv_shift) - 1));
            }
        }
        places[i] = p;
    }
    __syncthreads();
}

template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t elem, float (&x)[8]) {
    const T* p = static_cast<const T*>(base) + elem;
    if constexpr (sizeof(T) == 2) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                x[2 * e] = f.x;
                x[2 * e + 1] = f.y;
            } else {
                x[2 * e] = __uint_as_float(w[e] << 16);
                x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    } else {
        const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    }
}

// Rotates a row of which this lane (of 16) holds the values 8 l .. 8 l + 7.  All lanes of the warp.
__device__ __forceinline__ void rotate8(float (&x)[8], int64_t pos, int l, const Q8Launch& a) {
    if (a.neox) {               // pairs (d, d + 64): the partner sits 8 lanes away
        const int64_t i = pos * 64 + 8 * (l & 7);
        float c[8], n[8];
        load8<float>(a.rope_cs, i, c);
        load8<float>(a.rope_sn, i, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = __shfl_xor_sync(0xffffffffu, x[e], 8);
            x[e] = l < 8 ? __fmaf_rn(x[e], c[e], -__fmul_rn(y, n[e])) : __fmaf_rn(y, n[e], __fmul_rn(x[e], c[e]));
        }
    } else {
        const float4 c = *reinterpret_cast<const float4*>(a.rope_cs + pos * 64 + 4 * l), n = *reinterpret_cast<const float4*>(a.rope_sn + pos * 64 + 4 * l);
        const float cc[4] = {c.x, c.y, c.z, c.w}, nn[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x0 = x[2 * e], x1 = x[2 * e + 1];
            x[2 * e] = __fmaf_rn(x0, cc[e], -__fmul_rn(x1, nn[e]));
            x[2 * e + 1] = __fmaf_rn(x0, nn[e], __fmul_rn(x1, cc[e]));
        }
    }
}

template <int kFmt, typename T>
__global__ void __launch_bounds__(256) q8_append_kernel(Q8Launch a) {
    __shared__ Place places[kJobs];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, l = lane & 15;
    const int NKV = a.n_kv_heads, units = 2 * NKV + (a.q_rot ? a.n_heads : 0);
    const int64_t job0 = (int64_t)blockIdx.x * kJobs, jobs = (int64_t)a.n_tokens * units;
    const int tok0 = (int)(job0 / units);
    pdl_wait();
    float x[4][8];
    int tok[4], unit[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t job = job0 + 8 * warp + 2 * i + (lane >> 4);
        tok[i] = job < jobs ? (int)(job / units) : -1;
        unit[i] = job < jobs ? (int)(job - (int64_t)tok[i] * units) : 0;
        if (tok[i] >= 0) {
            const bool is_v = unit[i] >= NKV;
            if (unit[i] < 2 * NKV) load8<T>(is_v ? a.v : a.k, tok[i] * (is_v ? a.v_stride : a.k_stride) + (int64_t)(is_v ? unit[i] - NKV : unit[i]) * kHeadDim + 8 * l, x[i]);
            else load8<float>(a.q_rot, ((int64_t)tok[i] * a.n_heads + unit[i] - 2 * NKV) * kHeadDim + 8 * l, x[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        }
    }
    q8_places(a, places, job0, units);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Place p = tok[i] >= 0 ? places[tok[i] - tok0] : Place{-1, -1, 0};
        const bool is_q = unit[i] >= 2 * NKV, is_v = !is_q && unit[i] >= NKV;
        bool real = p.pos >= 0;
        if (a.rope_cs) {
            if (real && !is_v && p.pos >= a.rope_rows) {
                real = false;
                if (l == 0) q8_flag(a, NOVA_ERR_INVALID);
            }
            const bool turn = real && !is_v;
            if (__any_sync(0xffffffffu, turn)) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[i][e];
                rotate8(y, turn ? p.pos : 0, l, a);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (turn) x[i][e] = y[e];
            }
            float* const back = !turn ? nullptr : is_q ? a.q_rot + ((int64_t)tok[i] * a.n_heads + unit[i] - 2 * NKV) * kHeadDim
                                        : a.k_rot ? a.k_rot + ((int64_t)tok[i] * NKV + unit[i]) * kHeadDim : nullptr;
            if (back) {
                *reinterpret_cast<float4*>(back + 8 * l) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
                *reinterpret_cast<float4*>(back + 8 * l + 4) = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
            }
        }
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[i][e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (is_q || !real || p.page < 0) continue;
        amax = fmaxf(amax, kQ8MinAmax);
        const float inv = __fdiv_rn(q8_qmax<kFmt>(), amax);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(x[i][e], inv);
        const uint2 code = make_uint2(q8_encode4<kFmt>(make_float4(y[0], y[1], y[2], y[3])), q8_encode4<kFmt>(make_float4(y[4], y[5], y[6], y[7])));
        const int h = is_v ? unit[i] - NKV : unit[i];
        unsigned char* const pool = static_cast<unsigned char*>(is_v ? a.pool_v : a.pool_k);
        *reinterpret_cast<uint2*>(pool + (((p.page << a.kv_shift) + p.slot) * NKV + h) * kHeadDim + 8 * l) = code;
        if (l == 0) (is_v ? a.scale_v : a.scale_k)[((p.page * NKV + h) << a.kv_shift) + p.slot] = __fdiv_rn(amax, q8_qmax<kFmt>());
    }
}

template <int kFmt>
__global__ void __launch_bounds__(256) q8_read_kernel(Q8Launch a) {
    __shared__ Place places[kJobs];
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, l = lane & 15;
    const int NKV = a.n_kv_heads, units = 2 * NKV;
    const int64_t job0 = (int64_t)blockIdx.x * kJobs, jobs = (int64_t)a.n_tokens * units;
    const int tok0 = (int)(job0 / units);
    pdl_wait();
    q8_places(a, places, job0, units);
    uint2 code[4];
    float scale[4];
    int64_t dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t job = job0 + 8 * warp + 2 * i + (lane >> 4);
        dst[i] = -1;
        if (job >= jobs) continue;
        const int tok = (int)(job / units), unit = (int)(job - (int64_t)tok * units);
        const Place p = places[tok - tok0];
        if (p.page < 0) continue;
        const bool is_v = unit >= NKV;
        const int h = is_v ? unit - NKV : unit;
        const unsigned char* const pool = static_cast<const unsigned char*>(is_v ? a.pool_v : a.pool_k);
        code[i] = __ldg(reinterpret_cast<const uint2*>(pool + (((p.page << a.kv_shift) + p.slot) * NKV + h) * kHeadDim + 8 * l));
        scale[i] = __ldg((is_v ? a.scale_v : a.scale_k) + ((p.page * NKV + h) << a.kv_shift) + p.slot);
        dst[i] = ((int64_t)tok * NKV + h) * kHeadDim + 8 * l;
        if (is_v) dst[i] |= (int64_t)1 << 62;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (dst[i] < 0) continue;
        void* const out = dst[i] >> 62 ? a.v_out : a.k_out;
        const int64_t at = dst[i] & (((int64_t)1 << 62) - 1);
        const float4 x = q8_decode4<kFmt>(code[i].x), y = q8_decode4<kFmt>(code[i].y);
        const float f = scale[i];
        const float v[8] = {x.x * f, x.y * f, x.z * f, x.w * f, y.x * f, y.y * f, y.z * f, y.w * f};
        if (a.io == NOVA_IO_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(static_cast<float*>(out) + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (a.io == NOVA_IO_F16) {
                    w[e] = pack_h2(v[2 * e], v[2 * e + 1]);
                } else {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                    w[e] = *reinterpret_cast<const uint32_t*>(&b);
                }
            }
            *reinterpret_cast<uint4*>(static_cast<unsigned char*>(out) + 2 * at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15u) != 0; }

// Descriptors -> launch description, with every check that the host can make.
int q8_fill(const nova_q8_cache* c, const nova_q8_rows* r, Q8Launch& a) {
    if (!c || !r) return NOVA_ERR_INVALID;
    const nova_kv_shape& sh = c->shape;
    if (sh.kv_dtype != NOVA_KV_I8 && sh.kv_dtype != NOVA_KV_E4M3) return NOVA_ERR_UNSUPPORTED;
    if (sh.head_dim != kHeadDim || kv_shift_of_block(sh.kv_block) < 0) return NOVA_ERR_UNSUPPORTED;
    if (sh.n_heads <= 0 || sh.n_kv_heads <= 0 || sh.n_heads % sh.n_kv_heads) return NOVA_ERR_INVALID;
    if (sh.n_heads / sh.n_kv_heads > 128) return NOVA_ERR_UNSUPPORTED;
    if (c->layer < 0 || c->nb <= 0 || c->table_stride <= 0 || !c->pool_k || !c->pool_v || !c->scale_k || !c->scale_v || !c->tables) return NOVA_ERR_INVALID;
    if (misaligned(c->pool_k) || misaligned(c->pool_v) || misaligned(c->scale_k) || misaligned(c->scale_v)) return NOVA_ERR_INVALID;
    if (!c->rope_cs != !c->rope_sn || (c->rope_cs && c->rope_rows <= 0) || misaligned(c->rope_cs) || misaligned(c->rope_sn)) return NOVA_ERR_INVALID;
    if (((int64_t)c->layer + 1) * c->nb * sh.kv_block > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;      // slot rows are 32-bit coordinates
    if (r->io_dtype != NOVA_IO_F32 && r->io_dtype != NOVA_IO_F16 && r->io_dtype != NOVA_IO_BF16) return NOVA_ERR_UNSUPPORTED;
    if (r->n_sessions < 0 || r->n_tokens < 0 || r->max_tokens < 0 || (r->n_sessions > 0 && !r->n_past)) return NOVA_ERR_INVALID;
    if (!r->tok_start && r->n_sessions > 0 && (r->n_tokens % r->n_sessions || r->max_tokens != r->n_tokens / r->n_sessions)) return NOVA_ERR_INVALID;
    if (r->tok_start && r->n_tokens > 0 && r->max_tokens < 1) return NOVA_ERR_INVALID;
    const int64_t unit = r->io_dtype == NOVA_IO_F32 ? 4 : 8;      // elements in 16 bytes
    const int64_t q_row = (int64_t)sh.n_heads * kHeadDim, kv_row = (int64_t)sh.n_kv_heads * kHeadDim;
    auto stride_ok = [&](int64_t s, int64_t row) { return s == 0 || (s >= row && s % unit == 0); };
    if (!stride_ok(r->q_stride, q_row) || !stride_ok(r->out_stride, q_row) || !stride_ok(r->k_stride, kv_row) || !stride_ok(r->v_stride, kv_row))
        return NOVA_ERR_INVALID;
    std::memset(&a, 0, sizeof(a));
    a.pool_k = c->pool_k; a.pool_v = c->pool_v; a.scale_k = c->scale_k; a.scale_v = c->scale_v;
    a.tables = c->tables; a.table_stride = c->table_stride; a.slice_ids = c->slice_ids;
    a.n_past = r->n_past; a.tok_start = r->tok_start;
    a.rope_cs = c->rope_cs; a.rope_sn = c->rope_sn; a.rope_rows = c->rope_rows;
    a.status = c->status;
    a.n_sessions = r->n_sessions; a.n_tokens = r->n_tokens; a.max_tokens = r->max_tokens;
    a.uniform_tokens = r->tok_start || !r->n_sessions ? 0 : r->n_tokens / r->n_sessions;
    a.q_stride = r->q_stride ? r->q_stride : q_row; a.out_stride = r->out_stride ? r->out_stride : q_row;
    a.k_stride = r->k_stride ? r->k_stride : kv_row; a.v_stride = r->v_stride ? r->v_stride : kv_row;
    a.io = r->io_dtype; a.fmt = sh.kv_dtype; a.neox = sh.rope_neox;
    a.layer = c->layer; a.nb = c->nb; a.n_heads = sh.n_heads; a.n_kv_heads = sh.n_kv_heads; a.kv_shift = kv_shift_of_block(sh.kv_block);
    return NOVA_OK;
}

}  // namespace

template <int kFmt>
static cudaError_t append_as(const Q8Launch& a, unsigned blocks, cudaStream_t s) {
    // A programmatic dependent of whatever comes before it: its CTAs are in place when that ends, and wait until then.
    if (a.io == NOVA_IO_F32) return launch_kernel_pdl(q8_append_kernel<kFmt, float>, dim3(blocks), dim3(256), 0, s, true, a);
    if (a.io == NOVA_IO_F16) return launch_kernel_pdl(q8_append_kernel<kFmt, __half>, dim3(blocks), dim3(256), 0, s, true, a);
    return launch_kernel_pdl(q8_append_kernel<kFmt, __nv_bfloat16>, dim3(blocks), dim3(256), 0, s, true, a);
}

int launch_q8_append(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    const int64_t blocks = ((int64_t)a.n_tokens * (2 * a.n_kv_heads + (a.q_rot ? a.n_heads : 0)) + kJobs - 1) / kJobs;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    const cudaError_t e = a.fmt == NOVA_KV_I8 ? append_as<NOVA_KV_I8>(a, (unsigned)blocks, s) : append_as<NOVA_KV_E4M3>(a, (unsigned)blocks, s);
    if (e != cudaSuccess) {
        set_cuda_error(e, "8-bit append launch");
        return NOVA_ERR_CUDA;
    }
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

int launch_q8_read(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    const int64_t blocks = ((int64_t)a.n_tokens * 2 * a.n_kv_heads + kJobs - 1) / kJobs;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    const cudaError_t e = a.fmt == NOVA_KV_I8 ? launch_kernel_pdl(q8_read_kernel<NOVA_KV_I8>, dim3((unsigned)blocks), dim3(256), 0, s, true, a)
                                              : launch_kernel_pdl(q8_read_kernel<NOVA_KV_E4M3>, dim3((unsigned)blocks), dim3(256), 0, s, true, a);
    if (e != cudaSuccess) {
        set_cuda_error(e, "8-bit read launch");
        return NOVA_ERR_CUDA;
    }
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

}  // namespace novab

using namespace novab;

extern "C" {

int nova_launch_q8_append(const nova_q8_cache* c, const nova_q8_rows* r, const void* k, const void* v, nova_stream_t s) {
    Q8Launch a;
    const int rc = q8_fill(c, r, a);
    if (rc != NOVA_OK) return rc;
    if (a.n_tokens == 0 || a.n_sessions == 0) return NOVA_OK;
    if (!k || !v || misaligned(k) || misaligned(v)) return NOVA_ERR_INVALID;
    a.k = k; a.v = v;
    return launch_q8_append(a, (cudaStream_t)s);
}

int nova_launch_q8_read(const nova_q8_cache* c, const nova_q8_rows* r, void* k_out, void* v_out, nova_stream_t s) {
    Q8Launch a;
    const int rc = q8_fill(c, r, a);
    if (rc != NOVA_OK) return rc;
    if (a.n_tokens == 0 || a.n_sessions == 0) return NOVA_OK;
    if (!k_out || !v_out || misaligned(k_out) || misaligned(v_out)) return NOVA_ERR_INVALID;
    a.k_out = k_out; a.v_out = v_out;
    return launch_q8_read(a, (cudaStream_t)s);
}

size_t nova_q8_workspace_bytes(const nova_kv_shape* sh, const nova_q8_rows* r) {
    if (!sh || !r || sh->n_heads <= 0 || sh->n_kv_heads <= 0 || sh->n_heads % sh->n_kv_heads || r->n_sessions < 0 || r->n_tokens < 0) return 0;
    return q8_work_bytes(sh->n_heads, sh->n_kv_heads, r->n_sessions, r->n_tokens, r->max_tokens);
}

static int q8_attn(const nova_q8_cache* c, const nova_q8_rows* r, const void* q, const void* k, const void* v, void* out, int window,
                   bool append, void* work, size_t work_bytes, nova_stream_t s) {
    Q8Launch a;
    int rc = q8_fill(c, r, a);
    if (rc != NOVA_OK) return rc;
    if (window < 0) return NOVA_ERR_INVALID;
    if (a.n_tokens == 0 || a.n_sessions == 0) return NOVA_OK;
    if (!q || !out || misaligned(q) || misaligned(out) || misaligned(work)) return NOVA_ERR_INVALID;
    const size_t need = nova_q8_workspace_bytes(&c->shape, r);
    if (need > 0 && (!work || work_bytes < need)) return NOVA_ERR_INVALID;
    a.q = q; a.out = out; a.window = window;
    a.part = static_cast<float*>(work);
    if (append) {
        if (!k || !v || misaligned(k) || misaligned(v)) return NOVA_ERR_INVALID;
        a.k = k; a.v = v;
        a.append = 1;
    }
    return launch_q8_attn(a, work_bytes, (cudaStream_t)s);
}

int nova_launch_q8_attn(const nova_q8_cache* c, const nova_q8_rows* r, const void* q, void* out, int window, void* work, size_t work_bytes,
                        nova_stream_t s) {
    return q8_attn(c, r, q, nullptr, nullptr, out, window, false, work, work_bytes, s);
}

int nova_launch_q8_append_attn(const nova_q8_cache* c, const nova_q8_rows* r, const void* q, const void* k, const void* v, void* out, int window,
                               void* work, size_t work_bytes, nova_stream_t s) {
    return q8_attn(c, r, q, k, v, out, window, true, work, work_bytes, s);
}

}  // extern "C"
