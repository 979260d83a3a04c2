// q8_common.cuh — what the kernels of the 8-bit paged cache share: the launch description, the rows of a session, the
// element types of activations and codes.
//
// The cache: value = code * scale.  Codes [layer][NB][page tokens][NKV][128], one byte each (int8, or e4m3); one fp32
// scale per (token, kv head) [layer][NB][NKV][page tokens], kv head major within a page so that the scales of one
// head's tile of keys are one contiguous piece.
#pragma once
#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <type_traits>

#include "mma_common.cuh"

namespace novab {

// A row that is all zeros (or nearly) still gets a positive scale: amax is taken to be at least this.
constexpr float kQ8MinAmax = 8.6736173798840355e-19f;      // 2^-60
// ... and attention takes a scale of V to be at least this, so that its logarithm and reciprocal are finite for pages
// that were never written (zeroed scales).  Codes up to 448 times it are below 1e-18.
constexpr float kQ8MinScale = 8.4703294725430034e-22f;     // 2^-70

// The softmax reference of a row moves only when a score outgrows it by more than kQ8Step (log2 units), so accumulators are
// rescaled rarely; weights are 2^kQ8Top times 2^(x - ref).  The largest is then 2^11 .. 2^15, inside fp16, and a weight
// keeps fp16's 11 bits down to 2^-25 of the reference (below: steps of 2^-35 of it).
constexpr float kQ8Step = 4.f, kQ8Top = 11.f;

constexpr int kQ8MaxPos = 0x7ff00000;      // the largest position: what is added to one stays inside 32 bits
constexpr int kQ8MaxCtas = 160;      // CTAs of an attention launch, one per SM (sizes the workspaces)

struct Q8Launch {
    void* pool_k;
    void* pool_v;
    float* scale_k;
    float* scale_v;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* slice_ids;     // nullptr: session s uses table s
    const int32_t* n_past;        // [S] position of the first row of each session
    const int32_t* tok_start;     // [S + 1] rows of session s: [tok_start[s], tok_start[s + 1]); nullptr: uniform_tokens each
    const void* q;                // [n_tokens][NH][128], io type, rows q_stride elements apart
    const void* k;                // [n_tokens][NKV][128]
    const void* v;
    void* out;                    // [n_tokens][NH][128]
    void* k_out;                  // read back: [n_tokens][NKV][128]
    void* v_out;
    float* q_rot;                 // append only (fp32 activations): rotate q / k in place as well, or nullptr
    float* k_rot;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const float* rope_cs;         // nullptr: q and k are taken as they are
    const float* rope_sn;
    int64_t rope_rows;
    int32_t* status;
    float* part;                  // workspace of the attention
    int32_t n_sessions, n_tokens, max_tokens, uniform_tokens;
    int32_t one_part;             // single tokens, fp32 or fp16 activations: q and the weights as one fp16 value instead of two parts
    int32_t io, fmt, neox;
    int32_t layer, nb, n_heads, n_kv_heads, kv_shift;
    int32_t window;
    int32_t keys_cap;             // attention: keys that a block table has entries for (none behind them is looked for)
    int32_t append;               // attention: write the (single) new token of every session on the way
};

#ifdef __CUDACC__

// Rows of session s, never outside [0, n_tokens) whatever tok_start holds.
__device__ __forceinline__ void q8_rows(const Q8Launch& a, int s, int& first, int& count) {
    if (!a.tok_start) {
        first = s * a.uniform_tokens;
        count = a.uniform_tokens;
        return;
    }
    int f = __ldg(a.tok_start + s), e = __ldg(a.tok_start + s + 1);
    f = f < 0 ? 0 : (f > a.n_tokens ? a.n_tokens : f);
    e = e < f ? f : (e > a.n_tokens ? a.n_tokens : e);
    first = f;
    count = e - f < a.max_tokens ? e - f : a.max_tokens;
}

// Session and token-within-session of row r: the last session that starts at or before r (-1: the row is nobody's).
__device__ __forceinline__ int q8_session_of(const Q8Launch& a, int r, int& t) {
    if (!a.tok_start) {
        const int s = r / a.uniform_tokens;
        t = r - s * a.uniform_tokens;
        return s < a.n_sessions ? s : -1;
    }
    int lo = 0, up = a.n_sessions;
    while (up - lo > 1) {
        const int mid = (lo + up) >> 1;
        if (__ldg(a.tok_start + mid) <= r) lo = mid; else up = mid;
    }
    int first, count;
    q8_rows(a, lo, first, count);
    t = r - first;
    return t >= 0 && t < count ? lo : -1;
}

__device__ __forceinline__ const int32_t* q8_table(const Q8Launch& a, int s) {
    return a.tables + (int64_t)(a.slice_ids ? __ldg(a.slice_ids + s) : s) * a.table_stride;
}

__device__ __forceinline__ void q8_flag(const Q8Launch& a, int code) {
    if (a.status) atomicCAS(a.status, 0, code);
}

// ---- activations: four consecutive values as fp32
template <typename T> struct Q8Io;
template <> struct Q8Io<float> {
    static __device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
    static __device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
};
template <> struct Q8Io<__half> {
    static __device__ __forceinline__ float4 load4(const __half* p) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    static __device__ __forceinline__ void store4(__half* p, float4 v) {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
template <> struct Q8Io<__nv_bfloat16> {
    static __device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    }
    static __device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
// The same with the type known only at run time (a few loads per row: the branch is uniform).
__device__ __forceinline__ float4 q8_load4(const void* base, int64_t elem, int io) {
    if (io == NOVA_IO_F32) return Q8Io<float>::load4(static_cast<const float*>(base) + elem);
    if (io == NOVA_IO_F16) return Q8Io<__half>::load4(static_cast<const __half*>(base) + elem);
    return Q8Io<__nv_bfloat16>::load4(static_cast<const __nv_bfloat16*>(base) + elem);
}
__device__ __forceinline__ void q8_store4(void* base, int64_t elem, int io, float4 v) {
    if (io == NOVA_IO_F32) Q8Io<float>::store4(static_cast<float*>(base) + elem, v);
    else if (io == NOVA_IO_F16) Q8Io<__half>::store4(static_cast<__half*>(base) + elem, v);
    else Q8Io<__nv_bfloat16>::store4(static_cast<__nv_bfloat16*>(base) + elem, v);
}

// Eight consecutive values (16 or 32 bytes), as loaded.
template <typename T>
__device__ __forceinline__ void q8_unpack8(const uint4* u, float (&x)[8]) {
    const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
    if constexpr (sizeof(T) == 2) {
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
        const uint32_t v[4] = {u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = __uint_as_float(w[e]);
            x[4 + e] = __uint_as_float(v[e]);
        }
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]), pack_h2(v[4], v[5]), pack_h2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- codes: four of them in a word
// Four codes of a word -> two pairs of fp16, exactly.
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

// The same over kQ8CodeDiv, exactly, for operands that are multiplied by a scale in fp16: the scale can be that many times as large, which
// keeps its two fp16 parts above the end of fp16's grid (2^-24).  int8: at no cost, a number whose exponent is six lower.  e4m3: one
// multiplication (as bit patterns, which are the codes over 256 as they stand, they took longer: 382 instead of 355 us for 8 x (301-512)
// tokens).
template <int kFmt> constexpr float kQ8CodeDiv = kFmt == NOVA_KV_I8 ? 64.f : 256.f;
template <int kFmt> __device__ __forceinline__ void q8_to_small_h2(uint32_t w, uint32_t& h0, uint32_t& h1) {
    __half2 x, y;
    if constexpr (kFmt == NOVA_KV_I8) {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x4c4c4c4cu, 0x4140), b = __byte_perm(u, 0x4c4c4c4cu, 0x4342);        // 16 + (128 + code) / 64
        const __half2 k = __halves2half2(__ushort_as_half(0x4c80), __ushort_as_half(0x4c80));      // 18
        x = __hsub2(*reinterpret_cast<const __half2*>(&a), k);
        y = __hsub2(*reinterpret_cast<const __half2*>(&b), k);
    } else {
        q8_to_h2<kFmt>(w, h0, h1);
        const __half2 k = __halves2half2(__ushort_as_half(0x1c00), __ushort_as_half(0x1c00));      // 2^-8
        x = __hmul2(*reinterpret_cast<const __half2*>(&h0), k);
        y = __hmul2(*reinterpret_cast<const __half2*>(&h1), k);
    }
    h0 = *reinterpret_cast<const uint32_t*>(&x);
    h1 = *reinterpret_cast<const uint32_t*>(&y);
}

// The same in fp32 (through fp16: a conversion of an integer takes the special-function units, a quarter of the rate).
template <int kFmt> __device__ __forceinline__ float4 q8_decode4(uint32_t w) {
    uint32_t h0, h1;
    q8_to_h2<kFmt>(w, h0, h1);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)), b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    return make_float4(a.x, a.y, b.x, b.y);
}
// Round to nearest, ties to even, in both formats.  |x| <= Q but for the rounding of the product; a NaN becomes code 0
// (int8) or NaN (e4m3).
template <int kFmt> __device__ __forceinline__ uint32_t q8_encode4(float4 x) {
    if constexpr (kFmt == NOVA_KV_I8) {
        auto code = [](float f) -> uint32_t {
            int c = __float2int_rn(f);
            c = c > 127 ? 127 : (c < -127 ? -127 : c);
            return (uint32_t)c & 0xffu;
        };
        return code(x.x) | (code(x.y) << 8) | (code(x.z) << 16) | (code(x.w) << 24);
    } else {
        uint32_t w;
        asm("{ .reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3; mov.b32 %0, {l, h}; }"
            : "=r"(w) : "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w));
        return w;
    }
}
template <int kFmt> __device__ __forceinline__ constexpr float q8_qmax() { return kFmt == NOVA_KV_I8 ? 127.f : 448.f; }

// ---- one row over a warp: lane i holds the values 4i .. 4i + 3
__device__ __forceinline__ float q8_amax(float4 x) {
    float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Rotates it for position pos, in the fused form of the append kernel (rope_append.cu).  All 32 lanes.
__device__ __forceinline__ float4 q8_rotate(float4 x, int64_t pos, int lane, const Q8Launch& a) {
    if (a.neox) {               // pairs (d, d + 64): the partner sits 16 lanes away
        const float4 y = make_float4(__shfl_xor_sync(0xffffffffu, x.x, 16), __shfl_xor_sync(0xffffffffu, x.y, 16),
                                     __shfl_xor_sync(0xffffffffu, x.z, 16), __shfl_xor_sync(0xffffffffu, x.w, 16));
        const int i = 4 * (lane & 15);
        const float4 c = *reinterpret_cast<const float4*>(a.rope_cs + pos * 64 + i), s = *reinterpret_cast<const float4*>(a.rope_sn + pos * 64 + i);
        if (lane < 16)
            return make_float4(__fmaf_rn(x.x, c.x, -__fmul_rn(y.x, s.x)), __fmaf_rn(x.y, c.y, -__fmul_rn(y.y, s.y)),
                               __fmaf_rn(x.z, c.z, -__fmul_rn(y.z, s.z)), __fmaf_rn(x.w, c.w, -__fmul_rn(y.w, s.w)));
        return make_float4(__fmaf_rn(y.x, s.x, __fmul_rn(x.x, c.x)), __fmaf_rn(y.y, s.y, __fmul_rn(x.y, c.y)),
                           __fmaf_rn(y.z, s.z, __fmul_rn(x.z, c.z)), __fmaf_rn(y.w, s.w, __fmul_rn(x.w, c.w)));
    }
    const float2 c = *reinterpret_cast<const float2*>(a.rope_cs + pos * 64 + 2 * lane), s = *reinterpret_cast<const float2*>(a.rope_sn + pos * 64 + 2 * lane);
    return make_float4(__fmaf_rn(x.x, c.x, -__fmul_rn(x.y, s.x)), __fmaf_rn(x.x, s.x, __fmul_rn(x.y, c.x)),
                       __fmaf_rn(x.z, c.y, -__fmul_rn(x.w, s.y)), __fmaf_rn(x.z, s.y, __fmul_rn(x.w, c.y)));
}

// ---- arithmetic and shared-memory access of the attention kernels
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

// int8 codes as (code + 128) 2^-24, an fp16 subnormal whose bits are the byte.
__device__ __forceinline__ void q8_k_to_h2(uint32_t w, uint32_t& h0, uint32_t& h1) {
    const uint32_t u = w ^ 0x80808080u;
    h0 = __byte_perm(u, 0u, 0x4140);
    h1 = __byte_perm(u, 0u, 0x4342);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float lds_f1(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory"); }
__device__ __forceinline__ void sts_f1(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, float4 v) {
    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Transpose of an 8 x 8 matrix of 16-bit values over the warp (lane 4 r + c holds row r, columns 2c and 2c + 1).
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

#endif  // __CUDACC__

// Lets a kernel have `bytes` of dynamic shared memory on the current device, and sees that it is launched with the `regs` registers a
// thread that its roles share out (with fewer they would wait for good); asked of the driver once per kernel and device.
template <auto kKernel>
inline cudaError_t q8_allow_smem(int bytes, int regs = 0) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (bit & done.load(std::memory_order_relaxed)) return cudaSuccess;
    if (regs > 0) {
        cudaFuncAttributes at;
        e = cudaFuncGetAttributes(&at, kKernel);
        if (e != cudaSuccess) return e;
        if (at.numRegs < regs) return cudaErrorInvalidConfiguration;
    }
    e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// q8_cache.cu, q8_attn.cu (single tokens), q8_chunk.cu (everything else)
int launch_q8_append(const Q8Launch& a, cudaStream_t s);
int launch_q8_read(const Q8Launch& a, cudaStream_t s);
int launch_q8_attn(const Q8Launch& a, cudaStream_t s);
bool q8_is_decode(int n_heads, int n_kv_heads, int max_tokens);      // single tokens, at most 8 query heads per kv head: q8_attn.cu's kernel
int launch_q8_chunk(const Q8Launch& a, cudaStream_t s);
size_t q8_chunk_work_bytes(int n_heads, int n_kv_heads, int max_tokens);
size_t q8_work_bytes(int n_heads, int n_kv_heads, int n_sessions, int n_tokens, int max_tokens);

}  // namespace novab
