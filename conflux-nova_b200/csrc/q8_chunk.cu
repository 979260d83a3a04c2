// q8_chunk.cu — attention of chunks of new tokens over the 8-bit paged cache: a ragged number of tokens per session (drafted
// tokens, prompt chunks), causal or in a sliding window; also single tokens with more than 8 query heads per kv head.
//
// What bounds it: few rows over long contexts, HBM (264 bytes per key and kv head); many rows, the tensor cores and the
// exponentials (4 * 128 flops and one exponential per (query head, key)).
//
//   * tcgen05 with accumulators in tensor memory.  The (token, head) pairs that share a kv head are the rows of a tile: one
//     half of 128 rows (held twice, for alternate tiles), or two halves that share every K/V tile.  A unit of work is (session, kv head, tile of tokens); the 64-key tiles
//     of all units form one line that is dealt out evenly over one CTA per SM, so neither short sessions, nor long ones, nor
//     the causal triangle leave SMs idle.  Units that several CTAs worked on are merged by the kernel behind it.
//   * Twenty warps: 8 softmax (thread = row), 2 issuing MMAs (one per half), 8 converting, each of which brings in its own keys'
//     codes and scales, one that walks the line (and one idle).  The pipe runs on from one unit to the next.
//   * The tensor cores want fp16 operands, so a tile's codes become fp16 VALUES in shared memory, code times scale, in the
//     128-byte-swizzle layout that is the K-major form for S = Q.K^T and the MN-major form for O += P.V.  A scale (K's over 2;
//     q is multiplied by 2 / sqrt(128) log2 e) goes in as two fp16 parts, 64 or 256 times as large and the codes as much
//     smaller, and the product is rounded once: 2^-11; where fp16 has no more bits to give (its grid ends at 2^-24) 2^-23, of K 2^-22.
//     With exact codes as operands and the scales in the softmax instead, every thread had to read three floats per key
//     from shared memory, which took 1500 cycles of a 64-key tile.  So |K| saturates at 2^17 and |V| at 65504 here.
//     A lane's rows are chosen so that neither the reads (rows r and r ^ 5 side by side) nor the writes meet in a bank.
//   * q (rotated) and P are rounded to fp16; everything else is fp32.
//   * Measured (graph replay, append included; in calls on several states in turn): 2048 tokens over 16384, 40 / 8 heads, int8: 900 us =
//     810 TFLOP/s (917-936); 8 x (301-512) tokens over 2k-8k, e4m3: 355 us = 720 TFLOP/s (377); 16 x (0-8) tokens over 2k-8k, int8:
//     52 us = 1.5 TB/s (55); a window of 512, e4m3: 52-55 us (54).  A 64-key tile of 256 rows
//     takes some 2400 cycles.  The tensor cores are busy for 1020 of them, the special-function units for 1024; what sets the pace is
//     the softmax warps' own chain of some 300 dependent instructions per tile (two warps per scheduler; without the exponentials
//     it would still be 2200 or so).  A unit costs 5 us of q and 4 us of outputs beside its tiles.
//   * Every wait is bounded; tensor memory is released on every path.
#include "q8_common.cuh"
#include "tc5_common.cuh"

namespace novab {
namespace {

constexpr int kThreads = 640, kMergeThreads = 128;
// Registers a thread: at launch, and of the softmax, issuing and converting warps (120 / 64 / 88: 918 us for 2048 tokens over 16384,
// 128 / 64 / 80: 880, 136 / 48 / 80: 873, 144 / 48 / 72: the same).
constexpr int kRegsLaunch = 96, kRegsSoft = 136, kRegsIssue = 48, kRegsConv = 80;
static_assert(256 * kRegsSoft + 128 * kRegsIssue + 256 * kRegsConv <= kThreads * kRegsLaunch, "registers of the roles");
constexpr int kConv = 8;                              // converting warps
constexpr int kKeys = 64;                             // keys of a tile
constexpr int kHalfRows = 128;                        // rows of a half = M of the MMAs
constexpr int kSlab = kKeys * 128;                    // 64 rows x 128 B
constexpr int kQSlab = kHalfRows * 128;
constexpr int kRaw = 2;                               // tiles of its own (every other) that a converting warp has in flight
constexpr int kMasks = 8;                             // ring of "which keys exist", for the softmax
constexpr int kMaxSessions = 512;                     // sessions of one launch
constexpr int kOffK = 4 * kQSlab;                     // two fp16 K tiles (dims 0-63 | 64-127), two V tiles
constexpr int kOffV = kOffK + 2 * 2 * kSlab;
constexpr int kOffRaw = kOffV + 2 * 2 * kSlab;        // [converter][kRaw] 32 rows of codes
constexpr int kOffSc = kOffRaw + kConv * kRaw * 4096;    // [converter][kRaw] their scales
constexpr int kOffX = kOffSc + kConv * kRaw * 128;            // (m, l) of the second half's rows on their way to the first
constexpr int kOffPlan = kOffX + kHalfRows * 8;
struct ChunkPlan {
    long long line[kMaxSessions + 1];                 // where each session's tiles start on the line
    int first[kMaxSessions], count[kMaxSessions], past[kMaxSessions];
};
constexpr int kOffParts = kOffPlan + (int)((sizeof(ChunkPlan) + 15) / 16 * 16);
constexpr int kOffBar = kOffParts + 4 * 48;
constexpr int kSmem = kOffBar + 768;
static_assert(kSmem <= 232448, "shared memory of one CTA");
constexpr int kTmemCols = 512;                        // S of half h, buffer b: columns 128 h + 64 b (P over its first 32); O: 256 + 128 h
constexpr uint32_t kColO = 256;
constexpr float kKDiv = 2.f;                          // K goes in divided by this: magnitudes up to 2^17 (rotated fp16 keys fit), and q, multiplied
                                                      // by 0.255, the same
// As kQ8Step and kQ8Top (single tokens), but the reference moves less often, which costs more here (O rescaled in tensor
// memory): weights are 2^7 .. 2^15 at the largest, with fp16's 11 bits down to 2^-21 of the reference.
constexpr float kStep = 8.f, kTop = 7.f;
constexpr int kSetup = 8;                             // what a unit costs beside its tiles, in tiles (8 x (301-512) tokens: 2 362 us, 5 349, 8 340, 12 342)
constexpr int kFewTiles = 4;                          // token tiles that a thread counts for itself
constexpr int kMinTiles = 4;                          // a CTA gets at least that many
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kHalfRows >> 4) << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(kHeadDim >> 3) << 17) | ((uint32_t)(kHalfRows >> 4) << 24);

struct ChunkShape {
    int tq;              // tokens of a tile
    int dual;            // 0: the tile's rows are two halves that share every K/V tile; 1: at most 128 rows, both halves hold them
                         // and take every other K/V tile (few rows leave one half's softmax as the slowest step otherwise)
    int rows_cap;        // rows of a partial slot
};

// Tiles of a unit: keys [first16 * 16, keys_end) in steps of 64.
__device__ __forceinline__ int unit_first16(const Q8Launch& a, int past, int t0) {
    const int first = a.window > 0 && past + t0 - a.window + 1 > 0 ? past + t0 - a.window + 1 : 0;
    return first >> 4;
}
__device__ __forceinline__ int unit_tiles(const Q8Launch& a, int tq, int past, int count, int qt) {
    const int t1 = (qt + 1) * tq < count ? (qt + 1) * tq : count;
    const int end = past + t1 < a.keys_cap ? past + t1 : a.keys_cap;          // (keys behind the block table are not looked for)
    return max((((end + 15) >> 4) - unit_first16(a, past, qt * tq) + 3) >> 2, 1);
}

// All threads of the CTA; ends with __syncthreads().
__device__ inline void build_plan(const Q8Launch& a, const ChunkShape& sh, ChunkPlan& p, bool flag) {
    bool many = false;
    for (int s = (int)threadIdx.x; s < a.n_sessions; s += (int)blockDim.x) {
        int first, count;
        q8_rows(a, s, first, count);
        const int past = __ldg(a.n_past + s);
        if (count > 0 && (past < 0 || past > kQ8MaxPos - count)) {
            if (flag) q8_flag(a, NOVA_ERR_INVALID);
            count = 0;
        }
        if (flag && count > 0 && past + count > a.keys_cap) q8_flag(a, NOVA_ERR_BAD_TABLE);
        long long len = 0;
        if (count <= kFewTiles * sh.tq)
            for (int qt = 0; qt * sh.tq < count; ++qt) len += unit_tiles(a, sh.tq, past, count, qt) + kSetup;
        else
            many = true;                                  // (a thread for itself needs 40 cycles a token tile)
        p.line[s + 1] = len * a.n_kv_heads;
        p.first[s] = first;
        p.count[s] = count;
        p.past[s] = past;
    }
    if (__syncthreads_or(many)) {
        for (int s = (int)threadIdx.x >> 5; s < a.n_sessions; s += (int)blockDim.x >> 5) {
            const int count = p.count[s], past = p.past[s];
            if (count <= kFewTiles * sh.tq) continue;
            long long len = 0;
            for (int qt = (int)threadIdx.x & 31; qt * sh.tq < count; qt += 32) len += unit_tiles(a, sh.tq, past, count, qt) + kSetup;
#pragma unroll
            for (int o = 16; o; o >>= 1) len += __shfl_xor_sync(0xffffffffu, len, o);
            if ((threadIdx.x & 31) == 0) p.line[s + 1] = len * a.n_kv_heads;
        }
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        const int lane = (int)threadIdx.x;
        long long carry = 0;
        if (lane == 0) p.line[0] = 0;
        for (int base = 0; base < a.n_sessions; base += 32) {
            long long v = base + lane < a.n_sessions ? p.line[base + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long t = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += t;
            }
            if (base + lane < a.n_sessions) p.line[base + lane + 1] = carry + v;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}
__device__ __forceinline__ int plan_ctas(long long total, int grid) {
    const long long most = (total + kMinTiles - 1) / kMinTiles;
    return most < grid ? (int)most : grid;
}
// (a 64-bit division is a hundred instructions and more, and these are on the way to a CTA's first load)
__device__ __forceinline__ long long div_ll(long long x, long long y) {
    return ((unsigned long long)x | (unsigned long long)y) >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}
// Where CTA c begins: shares that differ by one at most.
struct Shares {
    long long each, more;      // the first `more` CTAs get one more than `each`
};
__device__ __forceinline__ Shares plan_shares(long long total, int n_ctas) {
    Shares s;
    s.each = div_ll(total, n_ctas);
    s.more = total - s.each * n_ctas;
    return s;
}
__device__ __forceinline__ long long cta_begin(const Shares& s, int c) { return c * s.each + (c < s.more ? c : s.more); }

struct Unit {
    int s, kvh, t0, t_cnt, past;     // session, kv head, first token of the tile, its tokens
    int first16, keys_end, tiles;
    long long begin, end;            // on the line, set-up weight included
};
// The unit at place pos of the line.  All lanes of a warp, same arguments.
__device__ inline Unit find_unit(const Q8Launch& a, const ChunkShape& sh, const ChunkPlan& p, long long pos) {
    const int lane = (int)threadIdx.x & 31;
    int lo = 0, up = a.n_sessions;
    while (up - lo > 1) {
        const int mid = (lo + up) >> 1;
        if (p.line[mid] <= pos) lo = mid; else up = mid;
    }
    while (lo + 1 < a.n_sessions && p.line[lo + 1] <= pos) ++lo;      // sessions without tiles
    Unit u;
    u.s = lo;
    u.past = p.past[lo];
    const int count = p.count[lo], nqt = (count + sh.tq - 1) / sh.tq;
    const long long off = pos - p.line[lo], per_head = div_ll(p.line[lo + 1] - p.line[lo], a.n_kv_heads);
    u.kvh = (int)div_ll(off, per_head);
    long long rem = off - u.kvh * per_head, base = 0;
    int qt = 0, len = 0;
    long long before = 0;
    for (int q0 = 0; q0 < nqt; q0 += 32) {
        const int v = q0 + lane < nqt ? unit_tiles(a, sh.tq, u.past, count, q0 + lane) + kSetup : 0;
        long long incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, rem < base + incl);
        if (hit) {
            const int l = __ffs(hit) - 1;
            qt = q0 + l;
            len = __shfl_sync(0xffffffffu, v, l);
            before = base + __shfl_sync(0xffffffffu, incl, l) - len;
            break;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    u.t0 = qt * sh.tq;
    u.t_cnt = count - u.t0 < sh.tq ? count - u.t0 : sh.tq;
    u.first16 = unit_first16(a, u.past, u.t0);
    u.keys_end = u.past + u.t0 + u.t_cnt;
    u.tiles = len - kSetup;
    u.begin = pos - rem + before;
    u.end = u.begin + len;
    return u;
}
// What the warps need to know of the part of a unit that their CTA works on.  One warp walks the line and leaves these in a ring; with
// the walk in every role the kernel was four times this code, and instruction fetches were its largest stall.
struct __align__(16) Part {
    int s, kvh, t0, t_cnt;
    int past, first16, keys_end, tile0;
    int tiles, whole, slot, pad;     // tiles 0: that was the last one; slot: which of the CTA's two partial slots
};
constexpr int kParts = 4;
static_assert(sizeof(Part) == 48 && kOffBar - kOffParts == kParts * (int)sizeof(Part), "ring of parts");
// The part [lo, hi) of the line that a CTA takes of the unit [begin, end), as tiles of the unit.
__device__ __forceinline__ void unit_part(long long begin, long long end, long long lo, long long hi, int& tile, int& count) {
    const long long b = (lo > begin ? lo : begin) - begin - kSetup, e = (hi < end ? hi : end) - begin - kSetup;
    tile = (int)(b > 0 ? b : 0);
    count = (int)(e > 0 ? e : 0) - tile;
    if (count < 0) count = 0;
}

// What the merge kernel needs of the unit that a CTA begins inside of; behind the partial slots.
struct __align__(16) Seam {
    long long begin, end;            // the unit on the line
    long long each, more;            // Shares
    int todo, c0, c_end;             // whether there is something to merge here; contributors c0 .. c_end - 1
    int token, t_cnt, pos, kvh, pad; // first row of q / out, rows, position of the first, kv head
};
static_assert(sizeof(Seam) == 64, "records of the seams");
__device__ __forceinline__ Seam* seams(const Q8Launch& a, const ChunkShape& sh) {
    return reinterpret_cast<Seam*>(a.part + (size_t)2 * kQ8MaxCtas * sh.rows_cap * kSlotW);
}

__device__ __forceinline__ unsigned long long pack_f2(float x, float y) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void unpack_f2(unsigned long long v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long add_f2(unsigned long long x, unsigned long long y) {
    unsigned long long v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}
template <int kRegs> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <int kFmt, typename T>
__global__ void __launch_bounds__(kThreads, 1)
q8_chunk_kernel(Q8Launch a, ChunkShape sh) {
    // No static shared memory: the dynamic region then starts at the front of the CTA's window, which is 1024-byte aligned as the
    // swizzled tiles need (checked).
    extern __shared__ unsigned char smem_raw[];
    ChunkPlan& plan = *reinterpret_cast<ChunkPlan*>(smem_raw + kOffPlan);
    uint32_t& s_tmem = *reinterpret_cast<uint32_t*>(smem_raw + kOffBar + 512);
    volatile int& s_abort = *reinterpret_cast<volatile int*>(smem_raw + kOffBar + 516);
    uint32_t* const s_mask = reinterpret_cast<uint32_t*>(smem_raw + kOffBar + 520);       // [kMasks][2] which keys of a tile exist
    uint32_t* const s_rmask = reinterpret_cast<uint32_t*>(smem_raw + kOffBar + 584);      // [kConv][kRaw] the same of a converter's 32 keys
    uint32_t* const s_show = reinterpret_cast<uint32_t*>(smem_raw + kOffBar + 648);       // ... whether what is no number among them shows
    const int lane = (int)threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int G = a.n_heads / a.n_kv_heads;
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bar = base + kOffBar;
    const uint32_t bar_partfull = bar, bar_partfree = bar + 32, bar_kfull = bar + 320, bar_kfree = bar + 336, bar_vfull = bar + 352, bar_vfree = bar + 368,
                   bar_sready = bar + 384 /* [half][buffer] */, bar_pready = bar + 416, bar_pvdone = bar + 448, bar_qready = bar + 480 /* [half] */,
                   bar_xfull = bar + 496, bar_xfree = bar + 504, bar_drain = bar + 712 /* [half] */;
    // Every waiter waits for a phase whose successor on the same barrier needs that waiter's own next action (or one that follows it),
    // so a parity is never taken for a later one.
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_kfull + 8u * i, kConv / 4);
            mbar_init(bar_kfree + 8u * i, sh.dual ? 1 : 2);
            mbar_init(bar_vfull + 8u * i, kConv / 4);
            mbar_init(bar_vfree + 8u * i, sh.dual ? 1 : 2);
            mbar_init(bar_qready + 8u * i, 4);
            mbar_init(bar_drain + 8u * i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar_sready + 8u * i, 1);
            mbar_init(bar_pready + 8u * i, 4);
            mbar_init(bar_pvdone + 8u * i, 1);
        }
        for (int i = 0; i < kParts; ++i) {
            mbar_init(bar_partfull + 8u * i, 1);
            mbar_init(bar_partfree + 8u * i, 18);      // every warp but the one that walks and the one that idles
        }
        mbar_init(bar_xfull, 4);
        mbar_init(bar_xfree, 4);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Nothing of the caller's is read before the kernels before this one are done, nor is the merge kernel let go, which reads
    // positions and row starts before its own wait.  Behind the append kernel only the cache itself is waited for (by the
    // converters): that kernel lets this one start once everything before it is done, and writes nothing else.
    if (!a.append) pdl_wait();
    pdl_launch_dependents();
    build_plan(a, sh, plan, blockIdx.x == 0);
    const long long total = plan.line[a.n_sessions];
    const int n_ctas = plan_ctas(total, (int)gridDim.x);
    if ((int)blockIdx.x >= n_ctas || (base & 1023u) != 0) {            // uniform over the CTA; nothing has been allocated yet
        if ((base & 1023u) != 0 && threadIdx.x == 0) q8_flag(a, NOVA_ERR_UNSUPPORTED);
        pdl_wait();                   // (a grid must not be done before the one that it follows)
        if (threadIdx.x == 0) seams(a, sh)[blockIdx.x].todo = 0;
        return;
    }
    const Shares shares = plan_shares(total, n_ctas);
    const long long lo = cta_begin(shares, (int)blockIdx.x), hi = cta_begin(shares, (int)blockIdx.x + 1);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"((uint32_t)kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    bool failed = false;
    int n = 0;                       // tiles of the parts before: every ring runs on over the parts
    Part* const ring = reinterpret_cast<Part*>(smem_raw + kOffParts);
    int k_part = 0;
    Part u;
    // The next part into u; false after the last one (or when a wait ran out).  All lanes of a warp.
    auto next_part = [&]() -> bool {
        const int slot = k_part & (kParts - 1);
        if (!__all_sync(0xffffffffu, t5_wait(bar_partfull + 8u * (uint32_t)slot, (uint32_t)(k_part / kParts) & 1u, &s_abort))) {
            failed = true;
            return false;
        }
        const int4* const src = reinterpret_cast<const int4*>(ring + slot);
        const int4 x = src[0], y = src[1], z = src[2];
        u.s = x.x; u.kvh = x.y; u.t0 = x.z; u.t_cnt = x.w;
        u.past = y.x; u.first16 = y.y; u.keys_end = y.z; u.tile0 = y.w;
        u.tiles = z.x; u.whole = z.y; u.slot = z.z;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_partfree + 8u * (uint32_t)slot);
        ++k_part;
        return u.tiles > 0;
    };

    if (warp < 8) {
        // ---------------------------------------------------------------------------------------- softmax: thread = one row
        regs_up<kRegsSoft>();
        const int half = warp >> 2, hrow = (int)threadIdx.x & (kHalfRows - 1);
        const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t col_s = 128u * (uint32_t)half, col_o = kColO + 128u * (uint32_t)half;
        const uint32_t my_sready = bar_sready + 16u * (uint32_t)half, my_pready = bar_pready + 16u * (uint32_t)half, my_pvdone = bar_pvdone + 16u * (uint32_t)half;
        const int row0 = sh.dual ? 0 : half * kHalfRows, row = row0 + hrow, tk = row / G, g = row - tk * G;
        const uint32_t per_g = (65536u + (uint32_t)G - 1u) / (uint32_t)G;       // rows / G by this: exact below 256 rows, G at most 128
        uint32_t xround = 0;
        auto arrive_warp = [&](uint32_t b) {                   // what all lanes have done so far
            __syncwarp();
            if (lane == 0) mbar_arrive(b);
        };
        while (!failed && next_part()) {
            const int tiles = u.tiles;
            // this half's tiles of the unit: every tile, or those whose place on the CTA's line is even (odd)
            const int mine0 = sh.dual ? (half + n) & 1 : 0, step = sh.dual ? 2 : 1;
            if (mine0 >= tiles) {
                n += tiles;
                continue;
            }
            const int64_t tok0 = (int64_t)plan.first[u.s] + u.t0;
            {
                // ---- q: rotated, scaled, fp16, K-major 128-byte swizzle; eight lanes a row, dims 8c .. and 64 + 8c .. each.  The scores
                // of the unit before are all computed (this thread has waited for the last of them), so the operand can be overwritten.
                // A warp takes four rows of every sixteen, two such groups at a time; the next two groups' q is on its way meanwhile (one
                // row after the other took 9 us a unit).
                constexpr float kQ = kAttnScale * kLog2e * kKDiv;
                constexpr int kRows = sizeof(T) == 4 ? 1 : 2, kVec = sizeof(T) / 2;
                const int c = lane & 7, second = a.neox ? 4 : 32;          // neox: the pairs (d, d + 64); else neighbours, in both halves of the dims
                const int rfirst = 4 * (warp & 3) + (lane >> 3), n_rows = u.t_cnt * G - row0;
                uint4 next[kRows][2 * kVec];
                auto bring = [&](int e8) {
#pragma unroll
                    for (int e = 0; e < kRows; ++e) {
                        const int rr = row0 + rfirst + 16 * (e8 + e), rt = (int)((uint32_t)rr * per_g >> 16), rg = rr - rt * G, rpos = u.past + u.t0 + rt;
#pragma unroll
                        for (int v = 0; v < 2 * kVec; ++v) next[e][v] = make_uint4(0u, 0u, 0u, 0u);
                        if (e8 < 8 && rt < u.t_cnt && !(a.rope_cs && rpos >= a.rope_rows)) {
                            const uint4* const src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (tok0 + rt) * a.q_stride + (int64_t)(u.kvh * G + rg) * kHeadDim + 8 * c);
#pragma unroll
                            for (int v = 0; v < kVec; ++v) {
                                next[e][v] = __ldg(src + v);
                                next[e][kVec + v] = __ldg(src + 8 * kVec + v);
                            }
                        }
                    }
                };
                bring(0);
#pragma unroll 1
                for (int e8 = 0; e8 < 8; e8 += kRows) {
                    const int r0 = rfirst + 16 * e8;
                    if (16 * e8 >= n_rows) {                               // none of these rows exists
#pragma unroll
                        for (int e = 0; e < kRows; ++e)
#pragma unroll
                            for (int hf = 0; hf < 2; ++hf)
                                sts128(base + (uint32_t)((2 * half + hf) * kQSlab + (r0 + 16 * e) * 128 + ((c ^ ((r0 + 16 * e) & 7)) << 4)), make_float4(0.f, 0.f, 0.f, 0.f));
                        continue;
                    }
                    uint4 raw[kRows][2 * kVec];
                    float4 rc[kRows][2], rs[kRows][2];
#pragma unroll
                    for (int e = 0; e < kRows; ++e) {
#pragma unroll
                        for (int v = 0; v < 2 * kVec; ++v) raw[e][v] = next[e][v];
#pragma unroll
                        for (int v = 0; v < 2; ++v) rc[e][v] = rs[e][v] = make_float4(0.f, 0.f, 0.f, 0.f);
                        const int rt = (int)((uint32_t)(row0 + r0 + 16 * e) * per_g >> 16), rpos = u.past + u.t0 + rt;
                        if (rt < u.t_cnt && a.rope_cs && rpos < a.rope_rows) {
                            const float* cr = a.rope_cs + (int64_t)rpos * 64 + (a.neox ? 8 : 4) * c;
                            const float* sr = a.rope_sn + (int64_t)rpos * 64 + (a.neox ? 8 : 4) * c;
                            rc[e][0] = __ldg(reinterpret_cast<const float4*>(cr));
                            rc[e][1] = __ldg(reinterpret_cast<const float4*>(cr + second));
                            rs[e][0] = __ldg(reinterpret_cast<const float4*>(sr));
                            rs[e][1] = __ldg(reinterpret_cast<const float4*>(sr + second));
                        }
                    }
                    bring(e8 + kRows);
#pragma unroll
                    for (int e = 0; e < kRows; ++e) {
                        const int r = r0 + 16 * e;
                        float x0[8], x1[8];
                        q8_unpack8<T>(&raw[e][0], x0);
                        q8_unpack8<T>(&raw[e][kVec], x1);
                        if (a.rope_cs) {
                            const float cc[8] = {rc[e][0].x, rc[e][0].y, rc[e][0].z, rc[e][0].w, rc[e][1].x, rc[e][1].y, rc[e][1].z, rc[e][1].w};
                            const float ss[8] = {rs[e][0].x, rs[e][0].y, rs[e][0].z, rs[e][0].w, rs[e][1].x, rs[e][1].y, rs[e][1].z, rs[e][1].w};
                            if (a.neox) {
#pragma unroll
                                for (int d = 0; d < 8; ++d) {
                                    const float y0 = x0[d], y1 = x1[d];
                                    x0[d] = __fmaf_rn(y0, cc[d], -__fmul_rn(y1, ss[d]));
                                    x1[d] = __fmaf_rn(y0, ss[d], __fmul_rn(y1, cc[d]));
                                }
                            } else {
#pragma unroll
                                for (int d = 0; d < 8; ++d) {
                                    float* y = d < 4 ? x0 : x1;
                                    const float y0 = y[2 * (d & 3)], y1 = y[2 * (d & 3) + 1];
                                    y[2 * (d & 3)] = __fmaf_rn(y0, cc[d], -__fmul_rn(y1, ss[d]));
                                    y[2 * (d & 3) + 1] = __fmaf_rn(y0, ss[d], __fmul_rn(y1, cc[d]));
                                }
                            }
                        }
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const uint32_t dst = base + (uint32_t)((2 * half + hf) * kQSlab + r * 128 + ((c ^ (r & 7)) << 4));
                            const float* y = hf ? x1 : x0;
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(pack_h2(y[0] * kQ, y[1] * kQ)), "r"(pack_h2(y[2] * kQ, y[3] * kQ)),
                                         "r"(pack_h2(y[4] * kQ, y[5] * kQ)), "r"(pack_h2(y[6] * kQ, y[7] * kQ))
                                         : "memory");
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive_warp(bar_qready + 8u * (uint32_t)half);
            }
            const int row_pos = u.past + u.t0 + tk;
            const bool in_tile = tk < u.t_cnt, beyond = in_tile && a.rope_cs && row_pos >= a.rope_rows;
            const bool row_ok = in_tile && !beyond;
            if (beyond && g == 0) q8_flag(a, NOVA_ERR_INVALID);
            // rows that are nobody's see everything: they never slow a warp down, and nothing of them is written
            const int row_lim = row_ok ? row_pos : 0x7fffffff;
            const int row_lo = row_ok && a.window > 0 ? row_pos - a.window + 1 : 0;
            const bool idle = __all_sync(0xffffffffu, !row_ok);
            // keys that all of the warp's rows see: [see_lo, see_hi]
            const int see_hi = __reduce_min_sync(0xffffffffu, row_lim), see_lo = __reduce_max_sync(0xffffffffu, row_lo);
            float m_ref = -INFINITY, l = 0.f;
            int m = sh.dual ? (n + mine0) >> 1 : n;            // tiles of this half so far: which score buffer, which parity
#pragma unroll 1
            for (int i = mine0; i < tiles; i += step, ++m) {
                const int t = n + i;
                if (!__all_sync(0xffffffffu, t5_wait(my_sready + 8u * (uint32_t)(m & 1), (uint32_t)(m >> 1) & 1u, &s_abort))) { failed = true; break; }
                if (idle) {                                     // what P and O hold in these rows is nobody's
                    arrive_warp(my_pready + 8u * (uint32_t)(m & 1));
                    continue;
                }
                tc_fence_after();
                const uint32_t s_col = t_lane + col_s + 64u * (uint32_t)(m & 1);
                const int key0 = (u.first16 << 4) + (u.tile0 + i) * kKeys;
                // All 64 scores in registers at once (read twice, 32 columns at a time, they took 12 % longer).
                uint32_t sv[2][32];
                tmem_ld32(s_col, sv[0]);
                tmem_ld32(s_col + 32u, sv[1]);
                const unsigned long long there = *reinterpret_cast<const unsigned long long*>(s_mask + 2 * (t & (kMasks - 1)));    // (a page missing, or the last key passed)
                tmem_wait_ld();
                if (key0 + kKeys - 1 > see_hi || key0 < see_lo || there != ~0ull) {
                    const int hi_k = row_lim - key0, lo_k = row_lo - key0;       // first and last visible column
                    unsigned long long vis = there;
                    if (hi_k < 63) vis &= hi_k < 0 ? 0ull : (2ull << hi_k) - 1ull;
                    if (lo_k > 0) vis &= lo_k > 63 ? 0ull : ~((1ull << lo_k) - 1ull);
                    const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
                    for (int c = 0; c < 32; ++c) {                             // -inf
                        if (!(v0 >> c & 1u)) sv[0][c] = 0xff800000u;
                        if (!(v1 >> c & 1u)) sv[1][c] = 0xff800000u;
                    }
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 2) m4[(c >> 1) & 3] = fmaxf(m4[(c >> 1) & 3], fmaxf(__uint_as_float(sv[c >> 5][c & 31]), __uint_as_float(sv[c >> 5][(c & 31) + 1])));
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                float scale = 1.f;
                if (mx > m_ref + kStep || (m_ref == -INFINITY && mx > -INFINITY)) {
                    scale = m_ref == -INFINITY ? 0.f : ex2(m_ref - mx);
                    m_ref = mx;
                }
                const float ms = m_ref == -INFINITY ? 0.f : kTop - m_ref;         // nothing visible yet: keep exp arguments finite
                const unsigned long long ms2 = pack_f2(ms, ms);
                unsigned long long sum2[2] = {0ull, 0ull};
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t pk[16];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float y0, y1;
                        unpack_f2(add_f2(pack_f2(__uint_as_float(sv[hf][c]), __uint_as_float(sv[hf][c + 1])), ms2), y0, y1);
                        y0 = ex2(y0);
                        y1 = ex2(y1);
                        sum2[(c >> 1) & 1] = add_f2(pack_f2(y0, y1), sum2[(c >> 1) & 1]);
                        pk[c >> 1] = pack_h2(y0, y1);
                    }
                    tmem_st16(s_col + 16u * (uint32_t)hf, pk);      // P over scores that have been read
                }
                float s0, s1;
                unpack_f2(add_f2(sum2[0], sum2[1]), s0, s1);
                l = fmaf(l, scale, s0 + s1);
                if (i > mine0 && __any_sync(0xffffffffu, scale != 1.f)) {
                    // O is rescaled between two P.V products: the previous one must be done
                    if (!__all_sync(0xffffffffu, t5_wait(my_pvdone + 8u * (uint32_t)((m - 1) & 1), (uint32_t)((m - 1) >> 1) & 1u, &s_abort))) { failed = true; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int cc = 0; cc < 4; ++cc) {
                        uint32_t ov[32];
                        tmem_ld32(t_lane + col_o + 32u * (uint32_t)cc, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * scale);
                        tmem_st32(t_lane + col_o + 32u * (uint32_t)cc, ov);
                    }
                    tmem_wait_st();
                }
                tmem_wait_st();
                tc_fence_before();
                arrive_warp(my_pready + 8u * (uint32_t)(m & 1));
            }
            n += tiles;
            if (failed) break;
            // ---- the unit's part is done: outputs, or a partial slot for the merge
            if (!__all_sync(0xffffffffu, t5_wait(my_pvdone + 8u * (uint32_t)((m - 1) & 1), (uint32_t)((m - 1) >> 1) & 1u, &s_abort))) { failed = true; break; }
            tc_fence_after();
            const bool whole = u.whole, fold = sh.dual && tiles > 1;
            const int xrows = sh.rows_cap <= 64 ? 64 : kHalfRows, xparts = sh.rows_cap <= 64 ? 1 : 2;       // rounds of handing over: all dims of 64 rows fit, or 64 of 128
            const uint32_t xbase = base + 2u * kQSlab, xml = base + kOffX;      // (the second half's q is no longer needed)
            if (fold && half == 1) {
                // both halves have a share of the rows: the second hands its own over, 64 dims at a time
                sts_f1(xml + 8u * (uint32_t)hrow, m_ref);
                sts_f1(xml + 8u * (uint32_t)hrow + 4u, l);
                for (int part = 0; part < xparts && !failed; ++part) {
#pragma unroll 1
                    for (int cc = 0; cc < 4 / xparts && !idle; ++cc) {
                        uint32_t ov[32];
                        tmem_ld32(t_lane + col_o + 64u * (uint32_t)part + 32u * (uint32_t)cc, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            sts128(xbase + (uint32_t)((8 * cc + (c >> 2)) * xrows + hrow) * 16u,
                                   make_float4(__uint_as_float(ov[c]), __uint_as_float(ov[c + 1]), __uint_as_float(ov[c + 2]), __uint_as_float(ov[c + 3])));
                    }
                    arrive_warp(bar_xfull);
                    if (!__all_sync(0xffffffffu, t5_wait(bar_xfree, xround & 1u, &s_abort))) failed = true;
                    ++xround;
                }
                tc_fence_before();
                continue;
            }
            const int64_t oe = (tok0 + tk) * a.out_stride + (int64_t)(u.kvh * G + g) * kHeadDim;
            // slot: (m, l) of every row, then the accumulators, four dims of every row side by side
            float* const slot = a.part + (size_t)(2 * blockIdx.x + u.slot) * ((size_t)sh.rows_cap * kSlotW);
            float w0 = 1.f, w1 = 0.f;                 // what this half's and the other half's accumulators are multiplied by
#pragma unroll 1
            for (int cc = 0; cc < 4; ++cc) {
                if (fold && (cc & (4 / xparts - 1)) == 0) {
                    if (!__all_sync(0xffffffffu, t5_wait(bar_xfull, xround & 1u, &s_abort))) { failed = true; break; }
                    ++xround;
                }
                if (cc == 0) {
                    if (fold) {
                        const float m1 = lds_f1(xml + 8u * (uint32_t)hrow), l1 = lds_f1(xml + 8u * (uint32_t)hrow + 4u);
                        const float mm = fmaxf(m_ref, m1);
                        w0 = m_ref == -INFINITY ? 0.f : ex2(m_ref - mm);
                        w1 = m1 == -INFINITY ? 0.f : ex2(m1 - mm);
                        l = l * w0 + l1 * w1;
                        m_ref = mm;
                    }
                    if (whole) {
                        const float inv = l > 0.f ? 1.f / l : 0.f;
                        w0 *= inv;
                        w1 *= inv;
                    } else if (row_ok) {
                        *reinterpret_cast<float2*>(slot + 2 * row) = make_float2(m_ref, l);
                    }
                }
                uint32_t ov[32];
                if (!idle) {
                    tmem_ld32(t_lane + col_o + 32u * (uint32_t)cc, ov);
                    tmem_wait_ld();
                }
                if (row_ok) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        float v[8];
#pragma unroll
                        for (int d = 0; d < 8; ++d) v[d] = __uint_as_float(ov[c + d]) * w0;
                        if (fold) {
#pragma unroll
                            for (int d = 0; d < 8; d += 4) {
                                const uint4 y = lds128(xbase + (uint32_t)((8 * (cc & (4 / xparts - 1)) + ((c + d) >> 2)) * xrows + hrow) * 16u);
                                v[d] = fmaf(__uint_as_float(y.x), w1, v[d]);
                                v[d + 1] = fmaf(__uint_as_float(y.y), w1, v[d + 1]);
                                v[d + 2] = fmaf(__uint_as_float(y.z), w1, v[d + 2]);
                                v[d + 3] = fmaf(__uint_as_float(y.w), w1, v[d + 3]);
                            }
                        }
                        if (whole) {
                            store8(static_cast<T*>(a.out) + oe + 32 * cc + c, v);
                        } else {
#pragma unroll
                            for (int d = 0; d < 8; d += 4)
                                *reinterpret_cast<float4*>(slot + 4 * (size_t)sh.rows_cap + ((size_t)(8 * cc + ((c + d) >> 2)) * sh.rows_cap + row) * 4) = make_float4(v[d], v[d + 1], v[d + 2], v[d + 3]);
                        }
                    }
                }
                if (fold && (cc & (4 / xparts - 1)) == 4 / xparts - 1) arrive_warp(bar_xfree);
            }
            tc_fence_before();
        }
    } else if (warp < 12) {
        regs_down<kRegsIssue>();
        if (warp < 10) {
            // ------------------------------------------------------------------------------------ MMA issue: one warp per half
            const int h = warp - 8;
            const uint32_t q_lo0 = umma_desc_lo(base + (uint32_t)(2 * h) * kQSlab, 16u), k_lo0 = umma_desc_lo(base + kOffK, 16u),
                           v_lo0 = umma_desc_lo(base + kOffV, (uint32_t)kSlab);
            const uint32_t col_s = tmem + 128u * (uint32_t)h, col_o = tmem + kColO + 128u * (uint32_t)h;
            // scores of tile t into this half's buffer m & 1
            auto issue_s = [&](int t, int m) -> bool {
                const uint32_t k_lo = k_lo0 + (uint32_t)(t & 1) * ((2 * kSlab) >> 4), d_s = col_s + 64u * (uint32_t)(m & 1);
                if (!__all_sync(0xffffffffu, t5_wait(bar_kfull + 8u * (uint32_t)(t & 1), (uint32_t)(t >> 1) & 1u, &s_abort))) return false;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        umma_f16(d_s, umma_desc_of(q_lo0 + (uint32_t)((j >> 2) * (kQSlab >> 4) + (j & 3) * 2)),
                                 umma_desc_of(k_lo + (uint32_t)((j >> 2) * (kSlab >> 4) + (j & 3) * 2)), kIdescS, j > 0 ? 1u : 0u);
                    umma_commit(bar_sready + 8u * (uint32_t)(2 * h + (m & 1)));
                    umma_commit(bar_kfree + 8u * (uint32_t)(t & 1));
                }
                __syncwarp();
                return true;
            };
            uint32_t seg = 0;
            while (!failed && next_part()) {
                const int tiles = u.tiles;
                const int mine0 = sh.dual ? (h + n) & 1 : 0, step = sh.dual ? 2 : 1;
                if (mine0 >= tiles) {
                    n += tiles;
                    continue;
                }
                int m = sh.dual ? (n + mine0) >> 1 : n;
                if (!__all_sync(0xffffffffu, t5_wait(bar_qready + 8u * (uint32_t)h, seg & 1u, &s_abort))) { failed = true; break; }
                ++seg;
                if (!issue_s(n + mine0, m)) { failed = true; break; }
                for (int i = mine0; i < tiles; i += step, ++m) {
                    const int t = n + i;
                    const uint32_t v_lo = v_lo0 + (uint32_t)(t & 1) * ((2 * kSlab) >> 4), p_col = col_s + 64u * (uint32_t)(m & 1);
                    // the scores of this half's next 64 keys first: they are computed while the softmax warps work on this tile
                    if (i + step < tiles && !issue_s(t + step, m + 1)) { failed = true; break; }
                    if (!__all_sync(0xffffffffu, t5_wait(bar_vfull + 8u * (uint32_t)(t & 1), (uint32_t)(t >> 1) & 1u, &s_abort))) { failed = true; break; }
                    if (!__all_sync(0xffffffffu, t5_wait(bar_pready + 8u * (uint32_t)(2 * h + (m & 1)), (uint32_t)(m >> 1) & 1u, &s_abort))) { failed = true; break; }
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            umma_f16_ts(col_o, p_col + (uint32_t)(8 * j), umma_desc_of(v_lo + (uint32_t)(j * (2048 >> 4))), kIdescPV, (j > 0 || i > mine0) ? 1u : 0u);
                        umma_commit(bar_pvdone + 8u * (uint32_t)(2 * h + (m & 1)));
                        umma_commit(bar_vfree + 8u * (uint32_t)(t & 1));
                    }
                    __syncwarp();
                }
                n += tiles;
            }
            if (failed) {
                // products that are under way finish before the tensor memory is given back (a bounded wait of its own)
                if (elect_one()) umma_commit(bar_drain + 8u * (uint32_t)h);
                __syncwarp();
                for (int i = 0; i < 1 << 16 && !mbar_try(bar_drain + 8u * (uint32_t)h, 0u); ++i) {}
                __syncwarp();
            }
        } else if (warp == 10) {
            // ------------------------------------------------------------------------------------ the walk along the line
            int k = 0;
            for (long long pos = lo;;) {
                Part q;
                q.tiles = 0;
                while (pos < hi && q.tiles == 0) {
                    const Unit v = find_unit(a, sh, plan, pos);
                    unit_part(v.begin, v.end, lo, hi, q.tile0, q.tiles);
                    pos = v.end;
                    q.s = v.s; q.kvh = v.kvh; q.t0 = v.t0; q.t_cnt = v.t_cnt; q.past = v.past; q.first16 = v.first16; q.keys_end = v.keys_end;
                    q.whole = q.tiles == v.tiles;
                    q.slot = v.begin > lo;
                }
                const int slot = k & (kParts - 1);
                if (k >= kParts && !__all_sync(0xffffffffu, t5_wait(bar_partfree + 8u * (uint32_t)slot, (uint32_t)(k / kParts - 1) & 1u, &s_abort))) { failed = true; break; }
                if (lane == 0) {
                    ring[slot] = q;
                    mbar_arrive(bar_partfull + 8u * (uint32_t)slot);
                }
                __syncwarp();
                ++k;
                if (q.tiles == 0) break;
            }
            // the unit that this CTA begins inside of is merged by its first such CTA, unless all its tiles went to one
            const Unit v = find_unit(a, sh, plan, lo);
            const int c1 = (int)blockIdx.x;
            Seam z = {};
            if (lo != v.begin && c1 > 0 && cta_begin(shares, c1 - 1) <= v.begin) {
                int c_end = c1, tile, some = 0;
                for (int c = c1 - 1, count; c < n_ctas && cta_begin(shares, c) < v.end; ++c) {
                    unit_part(v.begin, v.end, cta_begin(shares, c), cta_begin(shares, c + 1), tile, count);
                    some += count > 0;
                    c_end = c + 1;
                }
                z.begin = v.begin; z.end = v.end; z.each = shares.each; z.more = shares.more;
                z.todo = some > 1; z.c0 = c1 - 1; z.c_end = c_end;
                z.token = plan.first[v.s] + v.t0; z.t_cnt = v.t_cnt; z.pos = v.past + v.t0; z.kvh = v.kvh;
            }
            if (lane == 0) seams(a, sh)[c1] = z;
        }
    } else {
        // ---------------------------------------------------------------------------------------- codes -> fp16 operands
        // Four warps for K, four for V (V's buffer comes free only after the softmax of its tile, and the next K must not wait for
        // that); of the four, two take the even tiles and two the odd ones, 32 keys each.  A warp brings its codes and scales in itself,
        // kRaw tiles ahead, with 16-byte asynchronous copies into a ring of its own, which needs no barrier.  (As TMA boxes the rows of one
        // head are 2 KiB a copy, too little: one warp issuing all of a tile's copies took 1900 cycles a tile, eight warps with a box
        // and a run of scales each 900.  16 keys of every tile a warp: 1500 cycles a tile, most of it latency.)
        regs_down<kRegsConv>();
        const int me = warp - 12, which = me >> 2, par = me >> 1 & 1, hw = me & 1;
        const bool p8 = a.kv_shift == 3;
        const unsigned char* const pool = static_cast<const unsigned char*>(which ? a.pool_v : a.pool_k);
        const float* const scales = which ? a.scale_v : a.scale_k;
        const int lrow = lane >> 3, lch = lane & 7;        // this lane's rows (and + 4) and 16-byte piece of every copy
        const int slot_mask = (1 << a.kv_shift) - 1;
        // ---- what is copied next
        u.tiles = 0;
        const int32_t* table = nullptr;
        const unsigned char* pool_u = nullptr;             // rows of the part's kv head, this lane's row and piece
        const float* scale_u = nullptr;
        const uint32_t row_bytes = (uint32_t)a.n_kv_heads * kHeadDim, page_bytes = row_bytes << a.kv_shift, page_scales = (uint32_t)a.n_kv_heads << a.kv_shift;
        bool more = true, waited = !a.append;
        int c_i = 0, c_key = 0, c_own = 0, b0 = 0, b1 = 0, n0 = 0, n1 = 0, issued = 0;      // c_i, c_own: own tiles of the part, done and in all
        // block-table entry of the page that holds a key; -1: a bad one, -2: there is no such key, or none of an 8-token page is in the
        // window of any token (its entry may be gone)
        auto entry = [&](int key) -> int {
            if (key >= u.keys_end || (p8 && a.window > 0 && key + 8 <= u.past + u.t0 - a.window + 1)) return -2;
            const int64_t page = key >> a.kv_shift;
            if (page >= a.table_stride) return -1;
            const int e = __ldg(table + page);
            return e >= 0 && e < a.nb ? e : -1;
        };
        auto fetch = [&](int i) {                          // of own tiles i .. i + 15: lane = (tile, which 16 of its keys)
            n0 = n1 = -2;
            if (i + (lane >> 1) < c_own) {
                const int key = c_key + (i + (lane >> 1)) * 2 * kKeys + 16 * (lane & 1);
                n0 = entry(key);
                if (p8) n1 = entry(key + 8);
            }
        };
        const uint32_t raw0 = base + kOffRaw + (uint32_t)(me * kRaw * 4096), rsc0 = base + kOffSc + (uint32_t)(me * kRaw * 128);
        auto issue_next = [&]() {
            if (!more) return;
            while (c_i == c_own) {
                n += u.tiles;
                if (!next_part()) {
                    more = false;
                    return;
                }
                const int i0 = (par + n) & 1;
                c_i = 0;
                c_own = (u.tiles - i0 + 1) >> 1;
                table = q8_table(a, u.s);
                c_key = (u.first16 << 4) + (u.tile0 + i0) * kKeys + 32 * hw;
                const int64_t page0 = (int64_t)a.layer * a.nb;
                pool_u = pool + page0 * page_bytes + (uint32_t)(u.kvh * kHeadDim) + (uint32_t)lrow * row_bytes + 16u * (uint32_t)lch;
                scale_u = scales + page0 * page_scales + ((uint32_t)u.kvh << a.kv_shift) + 4 * (lane & 1);
                fetch(0);
            }
            if ((c_i & 15) == 0) {
                b0 = n0;
                b1 = n1;
                fetch(c_i + 16);
            }
            if (!waited) {
                pdl_wait();                                // the append before us has written the new rows (older keys too: another
                                                           // session of the call may have written them; not waiting gained nothing)
                waited = true;
            }
            const int key = c_key + c_i * 2 * kKeys;
            const uint32_t st = (uint32_t)(issued & (kRaw - 1)), dst = raw0 + st * 4096u + (uint32_t)(lrow * 128);
            int mine = 0;                                  // the entry behind key `lane`
#pragma unroll
            for (int g8 = 0; g8 < 4; ++g8) {               // eight rows each: one page of 8, or half of 16 slots
                int e = __shfl_sync(0xffffffffu, b0, (2 * c_i + (g8 >> 1)) & 31);
                if (p8) {
                    const int f = __shfl_sync(0xffffffffu, b1, (2 * c_i + (g8 >> 1)) & 31);
                    if (g8 & 1) e = f;
                }
                if (lrow == g8) mine = e;
                if (e >= 0) {
                    const int s0 = (key + 8 * g8) & slot_mask;
                    const unsigned char* src = pool_u + (uint64_t)(uint32_t)e * page_bytes + (uint32_t)s0 * row_bytes;
                    cp_async16(dst + (uint32_t)(g8 * 1024 + ((lch ^ lrow) << 4)), src);
                    cp_async16(dst + (uint32_t)(g8 * 1024 + 512 + ((lch ^ (lrow + 4)) << 4)), src + 4 * row_bytes);
                    if ((lane >> 1) == g8) cp_async16(rsc0 + st * 128u + (uint32_t)(16 * lane), scale_u + (uint64_t)(uint32_t)e * page_scales + s0);      // four keys a lane
                }
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, mine >= 0 && key + lane < u.keys_end);
            const bool bad = __any_sync(0xffffffffu, mine == -1);
            if (lane == 0) {
                s_rmask[me * kRaw + st] = mask;
                s_show[me * kRaw + st] = !which || (key + 31 <= u.past + u.t0 && (a.window <= 0 || key >= u.keys_end - a.window));
                if (bad && !which) q8_flag(a, NOVA_ERR_BAD_TABLE);
            }
            ++c_i;
            ++issued;
        };
        // ---- what is converted now.  Eight lanes share two rows that differ in bits 0 and 2: four 16-byte pieces of each, apart both
        // where they are read (piece c of row r sits at c ^ (r & 7)) and where they are written (pieces 2c and 2c + 1, likewise).
        const int r8 = (lane >> 3) ^ (5 * (lane >> 2 & 1)), c4 = lane & 3;
        const uint32_t bar_full = (which ? bar_vfull : bar_kfull) + 8u * (uint32_t)par, bar_free = (which ? bar_vfree : bar_kfree) + 8u * (uint32_t)par;
        const uint32_t dst0 = base + (which ? kOffV : kOffK) + (uint32_t)par * (2 * kSlab) + (uint32_t)(32 * hw + r8) * 128u;
        const float mul = kQ8CodeDiv<kFmt> * (which ? 1.f : 1.f / kKDiv);
        for (int k = 0; k < kRaw; ++k) {
            issue_next();
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
#pragma unroll 1
        for (int j = 0; j < issued; ++j) {                          // tile 2 j + par of the CTA's line
            asm volatile("cp.async.wait_group %0;" ::"n"(kRaw - 1) : "memory");      // (a group per tile, empty ones at the end)
            __syncwarp();
            if (j > 0 && !__all_sync(0xffffffffu, t5_wait(bar_free, (uint32_t)(j - 1) & 1u, &s_abort))) { failed = true; break; }
            const uint32_t st = (uint32_t)(j & (kRaw - 1)), mask = s_rmask[me * kRaw + st];
            if (!which && lane == 0) s_mask[2 * ((2 * j + par) & (kMasks - 1)) + hw] = mask;
            // What is no number stays none, so that it shows: the score of such a key is NaN for the queries that see it, and is taken out
            // for the others.  But V of a key that a query does not see is multiplied by zero: unless all the unit's queries see all of
            // these keys, it becomes the largest number.
            const bool show = s_show[me * kRaw + st];
            const __half2 most = __half2half2(__ushort_as_half(show ? 0x7fff : 0x7bff));            // (the minimum with NaN is the other)
            const uint32_t src = raw0 + st * 4096u + (uint32_t)r8 * 128u;
            // two rows (r8 and r8 + 8) at a time
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint4 code[4];                                      // dims of slab 0 and 1 of each
                float f[2];
#pragma unroll
                for (int e = 0; e < 4; ++e) code[e] = lds128(src + (uint32_t)(q * 2048 + (e >> 1) * 1024) + (((uint32_t)(4 * (e & 1) + c4) ^ (uint32_t)r8) << 4));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f[e] = lds_f1(rsc0 + st * 128u + (uint32_t)((16 * q + 8 * e + r8) * 4));
                    if (!(mask >> (16 * q + 8 * e + r8) & 1u)) {      // what does not exist may hold anything: zeros instead
                        code[2 * e] = code[2 * e + 1] = make_uint4(0u, 0u, 0u, 0u);
                        f[e] = 0.f;
                    }
                }
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    float fs = fminf(f[e2] * mul, 65504.f * kQ8CodeDiv<kFmt> / q8_qmax<kFmt>());
                    if (show) fs = fmaf(f[e2], 0.f, fs);              // (NaN for a scale that is no number)
                    const __half hi1 = __float2half_rn(fs);
                    const __half2 hi2 = __half2half2(hi1), lo2 = __half2half2(__float2half_rn(fs - __half2float(hi1)));
#pragma unroll
                    for (int e = 2 * e2; e < 2 * e2 + 2; ++e) {
                        uint32_t h[8];
                        q8_to_small_h2<kFmt>(code[e].x, h[0], h[1]);
                        q8_to_small_h2<kFmt>(code[e].y, h[2], h[3]);
                        q8_to_small_h2<kFmt>(code[e].z, h[4], h[5]);
                        q8_to_small_h2<kFmt>(code[e].w, h[6], h[7]);
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            const __half2 x = *reinterpret_cast<const __half2*>(&h[b]);
                            __half2 y = __hfma2(x, hi2, __hmul2(x, lo2));
                            if (kFmt == NOVA_KV_E4M3 && which) y = __hmin2(y, most);
                            h[b] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                        const uint32_t de = dst0 + (uint32_t)(q * 2048 + e2 * 1024 + (e & 1) * kSlab);
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(de + (((uint32_t)(2 * c4) ^ (uint32_t)r8) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(de + (((uint32_t)(2 * c4 + 1) ^ (uint32_t)r8) << 4)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_full);
            issue_next();                                           // into the stage that has just been read
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");           // nothing may land after the CTA is gone: no copy, and no arrival of the
        if (!failed && issued > 0) t5_wait(bar_free, (uint32_t)(issued - 1) & 1u, &s_abort);      // products of the last tiles either
    }
    if (failed && lane == 0) q8_flag(a, NOVA_ERR_TIMEOUT);
    // ---- release the tensor memory (every path of every thread ends here)
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemCols) : "memory");
}

// Merge of the units that several CTAs worked on, by the record of CTA blockIdx.x + 1.  blockIdx.y takes a share of the (32-row,
// 16-dim) pieces; thread = row, and what four contributors have for it is on its way at a time (with the loads one after the other, and
// the plan worked out again here, the merge took 42 us for 8 x (301-512) tokens).
__global__ void __launch_bounds__(kMergeThreads, 4) q8_chunk_merge_kernel(Q8Launch a, ChunkShape sh) {
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const int G = a.n_heads / a.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();                            // by every CTA: this grid must not be done before the one that it follows
    const int4* const rec = reinterpret_cast<const int4*>(seams(a, sh) + blockIdx.x + 1);
    int4 w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __ldcg(rec + e);
    const Seam z = *reinterpret_cast<const Seam*>(w);
    if (!z.todo) return;
    Shares shares;
    shares.each = z.each;
    shares.more = z.more;
    auto begin = [&](int c) -> long long { return cta_begin(shares, c); };
    const size_t slot_floats = (size_t)sh.rows_cap * kSlotW;
    const int rows = z.t_cnt * G, pieces = (rows + 31) / 32 * 8;
    for (int piece = (int)blockIdx.y * (kMergeThreads / 32) + warp; piece < pieces; piece += (int)gridDim.y * (kMergeThreads / 32)) {
        const int row = (piece >> 3) * 32 + lane, d4 = (piece & 7) * 4;
        const int tk = row / G, g = row - tk * G;
        if (row >= rows || (a.rope_cs && z.pos + tk >= a.rope_rows)) continue;
        float M = -INFINITY, L = 0.f;
        float4 acc[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = z.c0; c < z.c_end; c += 4) {
            float2 ml[4];
            float4 x[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ml[e] = make_float2(-INFINITY, 0.f);
                int tile, count = 0;
                if (c + e < z.c_end) unit_part(z.begin, z.end, begin(c + e), begin(c + e + 1), tile, count);
                if (count > 0) {
                    const float* slot = a.part + (size_t)(2 * (c + e) + (z.begin > begin(c + e) ? 1 : 0)) * slot_floats;
                    ml[e] = __ldcg(reinterpret_cast<const float2*>(slot + 2 * row));
#pragma unroll
                    for (int d = 0; d < 4; ++d) x[e][d] = __ldcg(reinterpret_cast<const float4*>(slot + 4 * (size_t)sh.rows_cap + ((size_t)(d4 + d) * sh.rows_cap + row) * 4));
                }
            }
            float mn = M;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (ml[e].y != 0.f) mn = fmaxf(mn, ml[e].x);
            const float cm = M == -INFINITY ? 0.f : ex2(M - mn);
            M = mn;
            L *= cm;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] = make_float4(acc[d].x * cm, acc[d].y * cm, acc[d].z * cm, acc[d].w * cm);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (ml[e].y == 0.f) continue;                 // nothing of the row's; a NaN stays one
                const float cx = ex2(ml[e].x - mn);
                L = fmaf(ml[e].y, cx, L);
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    acc[d] = make_float4(fmaf(x[e][d].x, cx, acc[d].x), fmaf(x[e][d].y, cx, acc[d].y), fmaf(x[e][d].z, cx, acc[d].z), fmaf(x[e][d].w, cx, acc[d].w));
            }
        }
        const float inv = L > 0.f ? 1.f / L : 0.f;
        const int64_t oe = ((int64_t)z.token + tk) * a.out_stride + (int64_t)(z.kvh * G + g) * kHeadDim + 4 * d4;
#pragma unroll
        for (int d = 0; d < 4; ++d) q8_store4(a.out, oe + 4 * d, a.io, make_float4(acc[d].x * inv, acc[d].y * inv, acc[d].z * inv, acc[d].w * inv));
    }
}

template <int kFmt, typename T>
cudaError_t launch_chunk_as(const Q8Launch& a, const ChunkShape& sh, int ctas, cudaStream_t s) {
    const cudaError_t e = q8_allow_smem<q8_chunk_kernel<kFmt, T>>(kSmem, kRegsLaunch);
    return e != cudaSuccess ? e : launch_kernel_pdl(q8_chunk_kernel<kFmt, T>, dim3((unsigned)ctas), dim3(kThreads), (size_t)kSmem, s, true, a, sh);
}
template <int kFmt>
cudaError_t launch_chunk(const Q8Launch& a, const ChunkShape& sh, int ctas, cudaStream_t s) {
    return a.io == NOVA_IO_F32 ? launch_chunk_as<kFmt, float>(a, sh, ctas, s)
         : a.io == NOVA_IO_F16 ? launch_chunk_as<kFmt, __half>(a, sh, ctas, s) : launch_chunk_as<kFmt, __nv_bfloat16>(a, sh, ctas, s);
}

ChunkShape chunk_shape(int n_heads, int n_kv_heads, int max_tokens) {
    ChunkShape sh;
    const int G = n_heads / n_kv_heads;
    const int64_t most = (int64_t)max_tokens * G;                       // rows of the longest chunk
    sh.dual = most <= kHalfRows;
    const int rows = sh.dual ? kHalfRows : 2 * kHalfRows;
    sh.tq = rows / G;
    sh.rows_cap = most < rows ? (int)((most + 31) / 32 * 32) : rows;
    return sh;
}

}  // namespace

size_t q8_chunk_work_bytes(int n_heads, int n_kv_heads, int max_tokens) {
    return (size_t)2 * kQ8MaxCtas * chunk_shape(n_heads, n_kv_heads, max_tokens).rows_cap * kSlotW * sizeof(float) + kQ8MaxCtas * sizeof(Seam);
}

int launch_q8_chunk(const Q8Launch& a, cudaStream_t s) {
    const ChunkShape sh = chunk_shape(a.n_heads, a.n_kv_heads, a.max_tokens);
    int ctas = sm_count();
    if (ctas > kQ8MaxCtas) ctas = kQ8MaxCtas;
    const size_t io_bytes = a.io == NOVA_IO_F32 ? 4 : 2;
    for (int s0 = 0; s0 < a.n_sessions; s0 += kMaxSessions) {           // (the plan's size)
        Q8Launch b = a;
        b.n_sessions = a.n_sessions - s0 < kMaxSessions ? a.n_sessions - s0 : kMaxSessions;
        b.n_past = a.n_past + s0;
        if (a.slice_ids) b.slice_ids = a.slice_ids + s0;
        else b.tables = a.tables + (int64_t)s0 * a.table_stride;
        if (s0 > 0) b.append = 0;          // (its rows are written: this launch comes after another attention, which waited for them)
        if (a.tok_start) {
            b.tok_start = a.tok_start + s0;
        } else {
            const int64_t rows = (int64_t)s0 * a.uniform_tokens;
            b.q = static_cast<const unsigned char*>(a.q) + rows * a.q_stride * (int64_t)io_bytes;
            b.out = static_cast<unsigned char*>(a.out) + rows * a.out_stride * (int64_t)io_bytes;
        }
        cudaError_t e = a.fmt == NOVA_KV_I8 ? launch_chunk<NOVA_KV_I8>(b, sh, ctas, s) : launch_chunk<NOVA_KV_E4M3>(b, sh, ctas, s);
        if (e == cudaSuccess) {
            count_launch();
            if (ctas > 1) e = launch_kernel_pdl(q8_chunk_merge_kernel, dim3((unsigned)ctas - 1, (unsigned)(sh.rows_cap / 16)), dim3(kMergeThreads), 0, s, true, b, sh);
        }
        if (e != cudaSuccess) {
            set_cuda_error(e, "8-bit chunk attention launch");
            return NOVA_ERR_CUDA;
        }
        NOVA_LAUNCH_CHECK();
    }
    return NOVA_OK;
}

}  // namespace novab
