// q8_cache.cu — writing the 8-bit paged cache and reading it back, and the C entry points of its operators.
//
// Writing: a row r (one token of one kv head; K rotated first where rotary tables are given, in the fused form of
// rope_append.cu) becomes  amax = max(max|r|, 2^-60),  scale = amax / Q,  code = rn(r * (Q / amax)),  Q = 127 (int8) or
// 448 (e4m3).  The three fp32 operations are rounded once each, so the codes are the same wherever the formula is followed.
// Reading: value = code * scale.
#include <cstring>

#include "q8_common.cuh"

namespace novab {
namespace {

// One warp per (row, head): heads [0, NKV) are K, [NKV, 2 NKV) V, and, when q is rotated in place too, the rest q.
template <int kFmt>
__global__ void __launch_bounds__(256) q8_append_kernel(Q8Launch a) {
    const int lane = (int)threadIdx.x & 31;
    const int NKV = a.n_kv_heads, units = 2 * NKV + (a.q_rot ? a.n_heads : 0);
    const int64_t job = (int64_t)blockIdx.x * 8 + ((int)threadIdx.x >> 5);
    if (job >= (int64_t)a.n_tokens * units) return;
    const int r = (int)(job / units), u = (int)(job - (int64_t)r * units);
    int t;
    const int s = q8_session_of(a, r, t);
    if (s < 0) return;
    const int64_t pos = (int64_t)__ldg(a.n_past + s) + t;
    const bool is_v = u >= NKV && u < 2 * NKV;
    const bool rot = a.rope_cs && !is_v;
    if (pos < 0 || (rot && pos >= a.rope_rows)) {
        if (lane == 0) q8_flag(a, NOVA_ERR_INVALID);
        return;
    }
    if (u >= 2 * NKV) {
        float* p = a.q_rot + ((int64_t)r * a.n_heads + (u - 2 * NKV)) * kHeadDim + 4 * lane;
        const float4 x = *reinterpret_cast<const float4*>(p);
        *reinterpret_cast<float4*>(p) = q8_rotate(x, pos, lane, a);
        return;
    }
    const int h = is_v ? u - NKV : u;
    float4 x = q8_load4(is_v ? a.v : a.k, (int64_t)r * (is_v ? a.v_stride : a.k_stride) + h * kHeadDim + 4 * lane, a.io);
    if (rot) {
        x = q8_rotate(x, pos, lane, a);
        if (a.k_rot) *reinterpret_cast<float4*>(a.k_rot + ((int64_t)r * NKV + h) * kHeadDim + 4 * lane) = x;
    }
    const int64_t lb = pos >> a.kv_shift;
    const int phys = lb < a.table_stride ? __ldg(q8_table(a, s) + lb) : -1;
    if (phys < 0 || phys >= a.nb) {
        if (lane == 0) q8_flag(a, NOVA_ERR_BAD_TABLE);
        return;
    }
    const float amax = fmaxf(q8_amax(x), kQ8MinAmax);
    const float inv = __fdiv_rn(q8_qmax<kFmt>(), amax);
    const uint32_t w = q8_encode4<kFmt>(make_float4(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv)));
    const int64_t page = (int64_t)a.layer * a.nb + phys;
    const int slot = (int)(pos & ((1 << a.kv_shift) - 1));
    unsigned char* pool = static_cast<unsigned char*>(is_v ? a.pool_v : a.pool_k);
    *reinterpret_cast<uint32_t*>(pool + (((page << a.kv_shift) + slot) * NKV + h) * kHeadDim + 4 * lane) = w;
    if (lane == 0) (is_v ? a.scale_v : a.scale_k)[((page * NKV + h) << a.kv_shift) + slot] = __fdiv_rn(amax, q8_qmax<kFmt>());
}

template <int kFmt>
__global__ void __launch_bounds__(256) q8_read_kernel(Q8Launch a) {
    const int lane = (int)threadIdx.x & 31;
    const int NKV = a.n_kv_heads;
    const int64_t job = (int64_t)blockIdx.x * 8 + ((int)threadIdx.x >> 5);
    if (job >= (int64_t)a.n_tokens * 2 * NKV) return;
    const int r = (int)(job / (2 * NKV)), u = (int)(job - (int64_t)r * 2 * NKV);
    int t;
    const int s = q8_session_of(a, r, t);
    if (s < 0) return;
    const int64_t pos = (int64_t)__ldg(a.n_past + s) + t;
    const int64_t lb = pos >> a.kv_shift;
    const int phys = pos >= 0 && lb < a.table_stride ? __ldg(q8_table(a, s) + lb) : -1;
    if (phys < 0 || phys >= a.nb) {
        if (lane == 0) q8_flag(a, NOVA_ERR_BAD_TABLE);
        return;
    }
    const bool is_v = u >= NKV;
    const int h = is_v ? u - NKV : u;
    const int64_t page = (int64_t)a.layer * a.nb + phys;
    const int slot = (int)(pos & ((1 << a.kv_shift) - 1));
    const unsigned char* pool = static_cast<const unsigned char*>(is_v ? a.pool_v : a.pool_k);
    const float4 c = q8_decode4<kFmt>(*reinterpret_cast<const uint32_t*>(pool + (((page << a.kv_shift) + slot) * NKV + h) * kHeadDim + 4 * lane));
    const float sc = (is_v ? a.scale_v : a.scale_k)[((page * NKV + h) << a.kv_shift) + slot];
    q8_store4(is_v ? a.v_out : a.k_out, ((int64_t)r * NKV + h) * kHeadDim + 4 * lane, a.io, make_float4(c.x * sc, c.y * sc, c.z * sc, c.w * sc));
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

int launch_q8_append(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    const int64_t blocks = ((int64_t)a.n_tokens * (2 * a.n_kv_heads + (a.q_rot ? a.n_heads : 0)) + 7) / 8;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    if (a.fmt == NOVA_KV_I8) q8_append_kernel<NOVA_KV_I8><<<(unsigned)blocks, 256, 0, s>>>(a);
    else q8_append_kernel<NOVA_KV_E4M3><<<(unsigned)blocks, 256, 0, s>>>(a);
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

int launch_q8_read(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    const int64_t blocks = ((int64_t)a.n_tokens * 2 * a.n_kv_heads + 7) / 8;
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    if (a.fmt == NOVA_KV_I8) q8_read_kernel<NOVA_KV_I8><<<(unsigned)blocks, 256, 0, s>>>(a);
    else q8_read_kernel<NOVA_KV_E4M3><<<(unsigned)blocks, 256, 0, s>>>(a);
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
