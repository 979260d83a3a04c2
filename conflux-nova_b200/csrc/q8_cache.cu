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

// A CTA takes kJobs consecutive (token, row) jobs, up to kIters times - a token's rows are its K heads, its V heads and, where q is
// rotated in place too, its query heads - a warp eight of them, eight lanes a row: lane c the values 8c .. 8c + 7 and 64 + 8c ..
// 64 + 8c + 7, so that both kinds of rotary pairs sit in one lane.  What the first rows hold is asked for before it is known
// where they go (session, position, page: a chain of dependent loads, one thread per token), so that one wait covers both; the
// rows of every later turn are on their way while the turn before is worked on.
// HBM should bound it (2 * 128 * (io bytes) read and 2 * 132 written per token and kv head); with 16 lanes a row, addresses in 64
// bits and two divisions in every lane the instructions did (1300 per warp: 253 MB in 141 us), with one turn per CTA the chain (87 us).
// Now 68 us = 3.7 TB/s for writing 16 x (1000-4096) tokens of 8 kv heads (253 MB) from bf16, 48 us = 5.3 TB/s for reading 256 MB back.
constexpr int kJobs = 64, kIters = 16;
struct Place {
    int64_t row;       // code row of kv head 0 in the pools, or -1: nowhere
    int64_t scale;     // scale of kv head 0
    int pos;           // position, or -1: nobody's row
};

constexpr int kStarts = 256;       // row starts kept in shared memory (more sessions: searched where they are)
struct PlaceSmem {
    Place places[kIters * kJobs / 2 + 2];      // (two rows a token at least)
    int starts[kStarts];
};

// The chain row starts -> (session) position and slice -> page is three round trips to memory.
__device__ __forceinline__ void q8_places(const Q8Launch& a, PlaceSmem& sm, int64_t job0, int jobs, int units) {
    const int tok0 = (int)(job0 / units);
    const int64_t last = (job0 + jobs - 1) / units;
    const int tok1 = last < a.n_tokens - 1 ? (int)last : a.n_tokens - 1;
    const bool staged = a.tok_start && a.n_sessions <= kStarts;
    if (staged) {
        for (int i = (int)threadIdx.x; i < a.n_sessions; i += (int)blockDim.x) sm.starts[i] = __ldg(a.tok_start + i);
        __syncthreads();
    }
    for (int i = (int)threadIdx.x; i <= tok1 - tok0; i += (int)blockDim.x) {
        Place p;
        p.row = p.scale = -1;
        p.pos = -1;
        int t, s;
        if (staged) {
            int lo = 0, up = a.n_sessions;
            while (up - lo > 1) {
                const int mid = (lo + up) >> 1;
                if (sm.starts[mid] <= tok0 + i) lo = mid; else up = mid;
            }
            int first, count;
            q8_rows(a, lo, first, count);
            t = tok0 + i - first;
            s = t >= 0 && t < count ? lo : -1;
        } else {
            s = q8_session_of(a, tok0 + i, t);
        }
        if (s >= 0) {
            const int64_t pos = (int64_t)__ldg(a.n_past + s) + t;
            const int32_t* const table = q8_table(a, s);
            if (pos < 0 || pos >= kQ8MaxPos) {
                q8_flag(a, NOVA_ERR_INVALID);
            } else {
                p.pos = (int)pos;
                const int64_t lb = pos >> a.kv_shift;
                const int phys = lb < a.table_stride ? __ldg(table + lb) : -1;
                if (phys >= 0 && phys < a.nb) {
                    const int64_t page = (int64_t)a.layer * a.nb + phys;
                    const int slot = (int)(pos & ((1 << a.kv_shift) - 1));
                    p.row = ((page << a.kv_shift) + slot) * a.n_kv_heads;
                    p.scale = ((page * a.n_kv_heads) << a.kv_shift) + slot;
                } else {
                    q8_flag(a, NOVA_ERR_BAD_TABLE);
                }
            }
        }
        sm.places[i] = p;
    }
    __syncthreads();
}

// Rotates a row of which this lane holds x0 (8c ..) and x1 (64 + 8c ..).
__device__ __forceinline__ void rotate16(float (&x0)[8], float (&x1)[8], int pos, int c, const Q8Launch& a) {
    const int64_t i = (int64_t)pos * 64 + (a.neox ? 8 : 4) * c;
    const int second = a.neox ? 4 : 32;           // neox: the pairs (d, d + 64); else neighbours, in both halves of the dims
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(a.rope_cs + i)), c1 = __ldg(reinterpret_cast<const float4*>(a.rope_cs + i + second));
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(a.rope_sn + i)), s1 = __ldg(reinterpret_cast<const float4*>(a.rope_sn + i + second));
    const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    if (a.neox) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y0 = x0[e], y1 = x1[e];
            x0[e] = __fmaf_rn(y0, cc[e], -__fmul_rn(y1, ss[e]));
            x1[e] = __fmaf_rn(y0, ss[e], __fmul_rn(y1, cc[e]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float* const y = e < 4 ? x0 : x1;
            const float y0 = y[2 * (e & 3)], y1 = y[2 * (e & 3) + 1];
            y[2 * (e & 3)] = __fmaf_rn(y0, cc[e], -__fmul_rn(y1, ss[e]));
            y[2 * (e & 3) + 1] = __fmaf_rn(y0, ss[e], __fmul_rn(y1, cc[e]));
        }
    }
}

// The job of lane group lane >> 3, half i, and the same of the next turn.
struct Job {
    int tok, unit;
    __device__ __forceinline__ void next(int units, int dt, int du) {      // kJobs = dt * units + du
        tok += dt;
        unit += du;
        if (unit >= units) {
            unit -= units;
            ++tok;
        }
    }
};

template <int kFmt, typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) q8_append_kernel(Q8Launch a, int iters) {
    constexpr int kVec = sizeof(T) / 2;           // 16-byte pieces of eight values
    __shared__ PlaceSmem sm;
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, c = lane & 7;
    const int NKV = a.n_kv_heads, units = 2 * NKV + (a.q_rot ? a.n_heads : 0);
    const int64_t job0 = (int64_t)blockIdx.x * kJobs * iters;
    const int tok0 = (int)(job0 / units), dt = kJobs / units, du = kJobs - dt * units;
    pdl_wait();
    pdl_launch_dependents();        // (a kernel that starts early reads nothing of the caller's that this one has not waited for)
    Job job[2];
    uint4 raw[2][2 * kVec];
    auto bring = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int v = 0; v < 2 * kVec; ++v) raw[i][v] = make_uint4(0u, 0u, 0u, 0u);
            if (job[i].tok >= a.n_tokens) continue;
            const int unit = job[i].unit;
            const bool is_v = unit >= NKV;
            const T* src;
            if (sizeof(T) == 4 && unit >= 2 * NKV) src = reinterpret_cast<const T*>(a.q_rot) + ((int64_t)job[i].tok * a.n_heads + unit - 2 * NKV) * kHeadDim;
            else src = static_cast<const T*>(is_v ? a.v : a.k) + job[i].tok * (is_v ? a.v_stride : a.k_stride) + (is_v ? unit - NKV : unit) * kHeadDim;
            const uint4* const p = reinterpret_cast<const uint4*>(src + 8 * c);
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                raw[i][v] = p[v];
                raw[i][kVec + v] = p[8 * kVec + v];
            }
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned j = (unsigned)(job0 - (int64_t)tok0 * units) + (unsigned)(8 * warp + 4 * i + (lane >> 3)), t = j / (unsigned)units;
        job[i].tok = tok0 + (int)t;
        job[i].unit = (int)(j - t * (unsigned)units);
    }
    bring();
    q8_places(a, sm, job0, kJobs * iters, units);
#pragma unroll 1
    for (int it = 0; it < iters; ++it) {
        float x0[2][8], x1[2][8], amax[2];
        Place p[2];
        int tok[2], unit[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            q8_unpack8<T>(&raw[i][0], x0[i]);
            q8_unpack8<T>(&raw[i][kVec], x1[i]);
            tok[i] = job[i].tok;
            unit[i] = job[i].unit;
            if (tok[i] < a.n_tokens) p[i] = sm.places[tok[i] - tok0];
            else p[i].row = p[i].pos = -1;
            job[i].next(units, dt, du);
        }
        if (it + 1 < iters) bring();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool is_q = unit[i] >= 2 * NKV, is_v = !is_q && unit[i] >= NKV;
            if (a.rope_cs && p[i].pos >= a.rope_rows) {              // (V's row too: the token is not written)
                p[i].row = -1;
                if (c == 0) q8_flag(a, NOVA_ERR_INVALID);
            } else if (a.rope_cs && p[i].pos >= 0 && !is_v) {
                rotate16(x0[i], x1[i], p[i].pos, c, a);
                float* const back = is_q ? a.q_rot + ((int64_t)tok[i] * a.n_heads + unit[i] - 2 * NKV) * kHeadDim
                                         : a.k_rot ? a.k_rot + ((int64_t)tok[i] * NKV + unit[i]) * kHeadDim : nullptr;
                if (back) {
                    store8(back + 8 * c, x0[i]);
                    store8(back + 64 + 8 * c, x1[i]);
                }
            }
            if (is_q) p[i].row = -1;
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaxf(fabsf(x0[i][e]), fabsf(x1[i][e])));
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            amax[i] = fmaxf(m, kQ8MinAmax);
        }
        // the divisions of the warp's eight rows in one go: lane c of a row takes amax[c & 1]
        const float am = c & 1 ? amax[1] : amax[0];
        const float inv_c = __fdiv_rn(q8_qmax<kFmt>(), am), scale_c = __fdiv_rn(am, q8_qmax<kFmt>());
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float inv = __shfl_sync(0xffffffffu, inv_c, (lane & 24) + i);
            if (p[i].row < 0) continue;
            const bool is_v = unit[i] >= NKV;
            const int h = is_v ? unit[i] - NKV : unit[i];
            float y0[8], y1[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y0[e] = __fmul_rn(x0[i][e], inv);
                y1[e] = __fmul_rn(x1[i][e], inv);
            }
            unsigned char* const dst = static_cast<unsigned char*>(is_v ? a.pool_v : a.pool_k) + (p[i].row + h) * kHeadDim + 8 * c;
            *reinterpret_cast<uint2*>(dst) = make_uint2(q8_encode4<kFmt>(make_float4(y0[0], y0[1], y0[2], y0[3])), q8_encode4<kFmt>(make_float4(y0[4], y0[5], y0[6], y0[7])));
            *reinterpret_cast<uint2*>(dst + 64) = make_uint2(q8_encode4<kFmt>(make_float4(y1[0], y1[1], y1[2], y1[3])), q8_encode4<kFmt>(make_float4(y1[4], y1[5], y1[6], y1[7])));
            if (c == i) (is_v ? a.scale_v : a.scale_k)[p[i].scale + ((int64_t)h << a.kv_shift)] = scale_c;
        }
    }
}

// Eight lanes a row: lane c the values 16 c .. 16 c + 15, a 16-byte load each.
template <int kFmt, typename T>
__global__ void __launch_bounds__(256) q8_read_kernel(Q8Launch a, int iters) {
    __shared__ PlaceSmem sm;
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5, c = lane & 7;
    const int NKV = a.n_kv_heads, units = 2 * NKV;
    const int64_t job0 = (int64_t)blockIdx.x * kJobs * iters;
    const int tok0 = (int)(job0 / units), dt = kJobs / units, du = kJobs - dt * units;
    pdl_wait();
    q8_places(a, sm, job0, kJobs * iters, units);
    Job job[2];
    uint4 code[2];
    float scale[2];
    T* dst[2];
    auto bring = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            dst[i] = nullptr;
            if (job[i].tok >= a.n_tokens) continue;
            const Place p = sm.places[job[i].tok - tok0];
            if (p.row < 0) continue;
            const bool is_v = job[i].unit >= NKV;
            const int h = is_v ? job[i].unit - NKV : job[i].unit;
            code[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(is_v ? a.pool_v : a.pool_k) + (p.row + h) * kHeadDim + 16 * c));
            scale[i] = __ldg((is_v ? a.scale_v : a.scale_k) + p.scale + ((int64_t)h << a.kv_shift));
            dst[i] = static_cast<T*>(is_v ? a.v_out : a.k_out) + ((int64_t)job[i].tok * NKV + h) * kHeadDim + 16 * c;
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned j = (unsigned)(job0 - (int64_t)tok0 * units) + (unsigned)(8 * warp + 4 * i + (lane >> 3)), t = j / (unsigned)units;
        job[i].tok = tok0 + (int)t;
        job[i].unit = (int)(j - t * (unsigned)units);
    }
    bring();
#pragma unroll 1
    for (int it = 0; it < iters; ++it) {
        uint4 now[2];
        float f[2];
        T* out[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            now[i] = code[i];
            f[i] = scale[i];
            out[i] = dst[i];
            job[i].next(units, dt, du);
        }
        if (it + 1 < iters) bring();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!out[i]) continue;
            const uint32_t w[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float4 x = q8_decode4<kFmt>(w[e]), y = q8_decode4<kFmt>(w[e + 1]);
                const float v[8] = {x.x * f[i], x.y * f[i], x.z * f[i], x.w * f[i], y.x * f[i], y.y * f[i], y.z * f[i], y.w * f[i]};
                store8(out[i] + 4 * e, v);
            }
        }
    }
}

bool misaligned(const void* p, unsigned to = 16) { return ((uintptr_t)p & (to - 1)) != 0; }

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
    if (misaligned(c->tables, 4) || misaligned(c->slice_ids, 4) || misaligned(c->status, 4) || misaligned(r->n_past, 4) || misaligned(r->tok_start, 4)) return NOVA_ERR_INVALID;
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
static cudaError_t append_as(const Q8Launch& a, unsigned blocks, int iters, cudaStream_t s) {
    // A programmatic dependent of whatever comes before it: its CTAs are in place when that ends, and wait until then.
    if (a.io == NOVA_IO_F32) return launch_kernel_pdl(q8_append_kernel<kFmt, float>, dim3(blocks), dim3(256), 0, s, true, a, iters);
    if (a.io == NOVA_IO_F16) return launch_kernel_pdl(q8_append_kernel<kFmt, __half>, dim3(blocks), dim3(256), 0, s, true, a, iters);
    return launch_kernel_pdl(q8_append_kernel<kFmt, __nv_bfloat16>, dim3(blocks), dim3(256), 0, s, true, a, iters);
}

template <int kFmt>
static cudaError_t read_as(const Q8Launch& a, unsigned blocks, int iters, cudaStream_t s) {
    if (a.io == NOVA_IO_F32) return launch_kernel_pdl(q8_read_kernel<kFmt, float>, dim3(blocks), dim3(256), 0, s, true, a, iters);
    if (a.io == NOVA_IO_F16) return launch_kernel_pdl(q8_read_kernel<kFmt, __half>, dim3(blocks), dim3(256), 0, s, true, a, iters);
    return launch_kernel_pdl(q8_read_kernel<kFmt, __nv_bfloat16>, dim3(blocks), dim3(256), 0, s, true, a, iters);
}

// CTAs, and turns of each: as many turns as leave every SM twelve CTAs (3: 134 us, 8: 118,
// 12: 115, 24: 129, 70 of one turn each: 156 us for writing 253 MB and reading as much).
static int64_t cache_blocks(int64_t jobs, int& iters) {
    const int64_t turns = (jobs + kJobs - 1) / kJobs, want = turns / (12 * sm_count());
    iters = (int)(want < 1 ? 1 : want > kIters ? kIters : want);
    return (turns + iters - 1) / iters;
}

int launch_q8_append(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    int iters;
    const int64_t blocks = cache_blocks((int64_t)a.n_tokens * (2 * a.n_kv_heads + (a.q_rot ? a.n_heads : 0)), iters);
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    const cudaError_t e = a.fmt == NOVA_KV_I8 ? append_as<NOVA_KV_I8>(a, (unsigned)blocks, iters, s) : append_as<NOVA_KV_E4M3>(a, (unsigned)blocks, iters, s);
    if (e != cudaSuccess) {
        set_cuda_error(e, "8-bit append launch");
        return NOVA_ERR_CUDA;
    }
    NOVA_LAUNCH_CHECK();
    return NOVA_OK;
}

int launch_q8_read(const Q8Launch& a, cudaStream_t s) {
    if (a.n_tokens <= 0 || a.n_sessions <= 0) return NOVA_OK;
    int iters;
    const int64_t blocks = cache_blocks((int64_t)a.n_tokens * 2 * a.n_kv_heads, iters);
    if (blocks > 0x7fffffffLL) return NOVA_ERR_TOO_LARGE;
    const cudaError_t e = a.fmt == NOVA_KV_I8 ? read_as<NOVA_KV_I8>(a, (unsigned)blocks, iters, s) : read_as<NOVA_KV_E4M3>(a, (unsigned)blocks, iters, s);
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
    return launch_q8_attn(a, (cudaStream_t)s);
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
