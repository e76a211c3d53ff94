// Prefill-chunk attention on the 5th-generation tensor cores (tcgen05 + TMEM) for the u8, f16 and (under bf16 activations)
// bf16 cache, head sizes 128 and 64.
//
// A work item is a q tile of 256 rows = (new token, q head of one GQA group) pairs of one
// (sequence, kv head), so a K/V byte is read once for the whole group.  The item is split into two
// halves A and B of 128 rows (UMMA M) that share the key / value operand tiles.  One persistent
// CTA per SM runs four roles that meet only through mbarriers:
//   loader    (1 thread)   TMA-engine bulk copies of the (block, head) records of 64-token tiles
//                          into a two-stage raw ring;
//   converter (4 warps)    raw bytes -> f16 operand tiles in 128-byte-swizzled layout:
//                          K' = byte * f16(k scale) as [64 tokens][128 dims], V'^T = byte *
//                          f16(v scale) as [128 dims][64 tokens] (the cache keeps value bytes
//                          token-minor, so both are K-major operands), two stages each;
//   mma       (one elected lane of a warp issues) tcgen05.mma: S_X = Q_X.K'^T into TMEM, O_X += P_X.V' in TMEM, for
//                          X = A, B.  u8 cache: one warp for both halves; as soon as half X has published P of tile j
//                          the S of tile j + 1 and then its P.V are queued, so the tensor core works on one half
//                          while the other half's softmax runs.  16-bit caches: a warp per half, S of tile j + 1
//                          queued as soon as the softmax warps hold S of tile j;
//   softmax   (2 x 4 warps) thread r owns row r of its half: reads S from TMEM, masks (diagonal
//                          tiles only), keeps a lazy running maximum, writes P = 2^(scale*(s-m)) as
//                          f16 into TMEM (the A operand of P.V); rescales O in TMEM only when a row maximum
//                          grew by more than 2^4; normalises and stores the output at the end.
// The zero-points ride on the tensor core: Q and K' carry 16 extra dims holding the row's sum of q
// and minus scale * zero-point split into f16 pieces, so S comes out with the offset term already
// subtracted; V'^T carries extra rows holding scale * zero-point (subtracted from O in the
// epilogue) and an all-ones row whose P.V column is the softmax denominator.
// The f16 cache needs no conversion: its four "converter" warps copy the token rows of a tile with
// 16-byte cp.async straight into the swizzled operand tiles (rows beyond the context are zero-filled).
// Key and value rows are both token-major there, so K' is a K-major operand and V' an MN-major one
// with the same shared-memory image; the softmax denominator comes from a second, 16-column P.V
// product against a constant tile whose first row is all ones.  The raw ring, the extra dims and
// the loader's copies do not exist in that variant.
// The CTA has four warpgroups (softmax A, softmax B, converter / copy, {mma, loader, second mma or idle, idle}) that re-divide the
// register file with setmaxnreg once their roles start: 160 registers per softmax thread, 104 per converter thread, 88 for
// the rest (one warp of each warpgroup shares a scheduler's 16 K registers).
// Every wait is bounded; a wait that runs out raises a flag that all roles poll.
// Masked steps (MK; include/masked_b200.h): a CTA has a slice of the q tiles' lists of context tiles (build_mask_items) and no counter; a tile of which a row
// sees a part takes that part from a word of bits; tokens that no row of the item sees go in as zeros and their blocks are not looked up; a piece
// leaves its rows' sums, maxima and unnormalised results to masked_join_kernel.  Few rows (one half's worth) are worked on by both halves, a tile each in
// turn.  The u8 cache has a warp for each half's products here too, S of a tile ahead of the P.V before it, and a pair of converter warps each for keys and
// values; the 16-bit caches' operand tiles are the loader's tensor copies, and the four warps beside it clear value rows that no row of the item sees.
// Tensor-bound for long contexts: 4 * Hq * D flops per (new token, context token) pair.
#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"
#include "tc05.cuh"

namespace pa {

namespace {

constexpr int kRows = 128;     // rows of one half = UMMA M
constexpr int kDx = 16;        // extra dims / extra V^T rows that carry the zero-point terms
constexpr int kKv = 64;        // context tokens per KV tile = UMMA N of Q.K^T
constexpr int kTmemCols = 512; // head size 128: S_A [0,64) S_B [64,128) O_A [128,272) O_B [272,416) P_A [416,448) P_B [448,480)
constexpr int kStages = 2;     // operand stages of the u8 variant (its raw ring has two more); the f16 variant has kStages16
constexpr int kStages16 = 4;
constexpr int kItemSlots = 4;   // depth of the queue that hands work items from the loader to the other roles
constexpr float kLazy = 4.f;   // log2 of the growth of a row maximum that forces a rescale of O
constexpr float kLog2eP = 1.4426950408889634f;
constexpr float kLn2P = 0.6931471805599453f;

constexpr int kSoftmaxWarps = 8, kConvWarps = 4;
constexpr int kWarpMma = kSoftmaxWarps + kConvWarps, kWarpLoad = kWarpMma + 1, kWarpMma2 = kWarpMma + 2;   // the second mma warp: 16-bit caches
constexpr int kThreads = 512;   // four warpgroups: softmax A, softmax B, converter / copy warps, {mma, loader, second mma (16-bit caches) or idle, idle}
// Registers per thread after the roles have re-divided the register file among the warpgroups (one warp of each shares a
// scheduler's 16 K registers: 160 + 160 + 104 + 88 = 512 x 32)
#ifndef PA_TC_REG_SOFTMAX
#define PA_TC_REG_SOFTMAX 160
#define PA_TC_REG_CONV 104
#define PA_TC_REG_MISC 88
#endif
template <int R> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
static_assert(kPrefillItemRows == 2 * kRows, "an item is two UMMA row tiles");

// One work item as every role sees it.
struct Item {
    int s, hk, t0, n_new, past;
    int row0;            // first (token, head) pair of half A
    int ctx_hi[2];       // context the last row of each half sees (0: the half has no rows)
    int nt[2];           // 64-token tiles of each half
    int ntiles;          // max of the two
    const int32_t* table;
};

// A masked step's item: tiles [j0, j0 + ntiles) of the q tile's list.  Where the q tile has rows for half A only, half B takes them too (`dup`): the
// halves take the tiles in turn, and half A joins both results.
struct MaskedItem : Item {
    VisTiles v;
    int lo;              // positions below it, beyond the sinks, are seen by no row
    int j0;
    int part;            // partial result, -1: the list is in one piece
    int tree, dup;
    __device__ __forceinline__ bool uses(int x, int j) const { return dup ? (j & 1) == x : j < nt[x]; }
    __device__ __forceinline__ int own(int j) const { return dup ? j >> 1 : j; }   // tile j among those of its half
};
template <bool MK> struct ItemOf { using type = Item; };
template <> struct ItemOf<true> { using type = MaskedItem; };

template <int BS, int CT, int D, bool MK>
struct PrefillSmem16;
template <int BS, int CT, int D, bool MK>
struct PrefillSmem;

template <int BS, int D, bool MK>
struct PrefillSmem<BS, PA_DTYPE_U8, D, MK> {
    static constexpr int NO = D + kDx;   // UMMA N of P.V
    static constexpr int NST = kStages;
    static constexpr int REC = BS * (D + 8);
    static constexpr int NREC = kKv / BS;
    static constexpr int RSTRIDE = REC + 64;       // records 64 bytes out of phase: conflict-free 16-byte reads across records
    alignas(1024) uint8_t q[2][kRows * D * 2];     // per half: D / 64 swizzle atoms of [128 rows][64 dims]
    alignas(1024) uint8_t k[kStages][kKv * D * 2];    // D / 64 atoms of [64 tokens][64 dims]
    alignas(1024) uint8_t vt[kStages][NO * kKv * 2];  // [D + 16 dims][64 tokens], groups of 8 rows
    alignas(128) uint8_t qx[2][kRows * kDx * 2];   // unswizzled [128 rows][16 dims]
    alignas(128) uint8_t kx[kStages][kKv * kDx * 2];  // unswizzled [64 tokens][16 dims]
    alignas(128) uint8_t raw_k[kStages][NREC * RSTRIDE];
    alignas(128) uint8_t raw_v[kStages][NREC * RSTRIDE];
    alignas(128) uint8_t out_stage[kSoftmaxWarps][32 * 128];   // 128 bytes of each of a warp's rows on their way to global memory
    alignas(16) uint2 v_tab[kConvWarps][kKv / 2];  // per converter warp: (scale, -1024 * scale) f16 pairs of two tokens
    alignas(16) uint2 tok_scale[MK ? kConvWarps : 1][MK ? kKv : 1];   // masked, per converter warp: a token's scale as the sum of two f16, each as a pair of equal ones
    alignas(8) uint64_t raw_full[kStages];   // loader -> converter (transaction bytes)
    alignas(8) uint64_t raw_free[kStages];   // converter -> loader
    alignas(8) uint64_t k_full[kStages];     // converter -> mma
    alignas(8) uint64_t v_full[kStages];
    alignas(8) uint64_t k_free[kStages];     // mma (commit) -> converter
    alignas(8) uint64_t v_free[kStages];
    alignas(8) uint64_t q_full[2];           // softmax -> mma, per item
    alignas(8) uint64_t s_full[2];           // mma (commit) -> softmax
    alignas(8) uint64_t s_read[2];           // softmax -> mma: S is in registers
    alignas(8) uint64_t p_full[2];           // softmax -> mma: P written, O rescaled
    alignas(8) uint64_t o_done[2];           // mma (commit) -> softmax: P.V complete
    alignas(8) uint64_t item_full[kItemSlots];   // loader -> every other warp
    alignas(8) uint64_t item_free[kItemSlots];   // every other warp -> loader: the slot has been read
    int item_ring[kItemSlots];
    typename ItemOf<MK>::type item_desc[kItemSlots];   // the loader locates an item once for every role
    alignas(8) uint64_t join_full, join_free;   // masked: half B -> half A: its rows' maxima and sums lie in its warps' out_stage; A -> B: it has read B's results
    uint32_t tmem_base;
    volatile int abort;
};

// f16 / bf16 cache: operand tiles only.  The bf16 variant has no denominator columns (P takes their place in tensor memory
// as two bf16 pieces, and the rows sum their own probabilities).
template <int BS, int D, bool MK>
struct PrefillSmem<BS, PA_DTYPE_F16, D, MK> : PrefillSmem16<BS, PA_DTYPE_F16, D, MK> {};
template <int BS, int D, bool MK>
struct PrefillSmem<BS, PA_DTYPE_BF16, D, MK> : PrefillSmem16<BS, PA_DTYPE_BF16, D, MK> {};

template <int BS, int CT, int D, bool MK>
struct PrefillSmem16 {
    static constexpr int NO = CT == PA_DTYPE_BF16 ? D : D + kDx;
    static constexpr int NREC = kKv / BS;
    static constexpr int NST = kStages16;
    alignas(1024) uint8_t q[2][kRows * D * 2];        // per half: D / 64 swizzle atoms of [128 rows][64 dims]
    alignas(1024) uint8_t k[NST][kKv * D * 2];    // D / 64 atoms of [64 tokens][64 dims], K-major
    alignas(1024) uint8_t vt[NST][kKv * D * 2];   // the same image read as an MN-major operand: atoms of 64 dims, 8-token groups 1024 bytes apart
    alignas(128) uint8_t out_stage[kSoftmaxWarps][32 * 128];
    alignas(128) uint8_t ones[16 * 16 * 2];           // unswizzled K-major [16 rows][16 tokens]: row 0 all ones
    alignas(8) uint64_t k_full[NST];     // copy warps -> mma (masked: the loader's copies)
    alignas(8) uint64_t v_full[NST];     // (masked: the warps that clear rows, of tiles that are not seen as a whole)
    alignas(8) uint64_t v_land[NST];     // masked: the loader's copies of values
    alignas(8) uint64_t k_free[NST];     // mma (commit) -> copy warps
    alignas(8) uint64_t v_free[NST];
    alignas(8) uint64_t q_full[2];
    alignas(8) uint64_t s_full[2];
    alignas(8) uint64_t s_read[2];
    alignas(8) uint64_t p_full[2];
    alignas(8) uint64_t o_done[2];
    alignas(8) uint64_t item_full[kItemSlots];
    alignas(8) uint64_t item_free[kItemSlots];
    int item_ring[kItemSlots];
    typename ItemOf<MK>::type item_desc[kItemSlots];   // the loader locates an item once for every role
    alignas(8) uint64_t join_full, join_free;   // masked: half B -> half A: its rows' maxima and sums lie in its warps' out_stage; A -> B: it has read B's results
    uint32_t tmem_base;
    volatile int abort;
};

__device__ __forceinline__ void cp_async16_zfill(void* dst_smem, const void* src_gmem, uint32_t src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst_smem)), "l"(src_gmem), "r"(src_bytes) : "memory");
}

__device__ __forceinline__ uint32_t sw128(uint32_t row, uint32_t chunk) { return row * 128u + ((chunk ^ (row & 7u)) << 4); }
// unswizzled K-major tile of 16 dims: 8-row groups 256 bytes apart, the two 8-dim halves 128 apart
__device__ __forceinline__ uint32_t plain16(uint32_t row, uint32_t half) { return (row >> 3) * 256u + half * 128u + (row & 7u) * 16u; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a, b) * s + t, two at a time
__device__ __forceinline__ float2 fma_pair(float a, float b, float s, float t) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a), "f"(b), "f"(s), "f"(t));
    return r;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ uint32_t ex2_h2(uint32_t x) {
    uint32_t y;
    asm("ex2.approx.f16x2 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t y;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
    return y;
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
__device__ __forceinline__ uint32_t hadd2_bits(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// f32 -> f16 through the packed conversion: the scalar form runs on the quarter-rate special
// function unit, which the softmax warps keep busy with exponentials
__device__ __forceinline__ __half f2h(float x) { return __ushort_as_half((unsigned short)(pack_h2(x, 0.f) & 0xffffu)); }
// z = h + m + l up to 2^-33 |z|, every piece an f16
__device__ __forceinline__ void split3(float z, __half& h, __half& m, __half& l) {
    h = f2h(z);
    const float r = z - __half2float(h);
    m = f2h(r);
    l = f2h(r - __half2float(m));
}
__device__ __forceinline__ uint32_t h2_bits(__half a, __half b) {
    return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}
// 16 cache bytes -> 16 f16 values 1024 + byte
__device__ __forceinline__ void bytes16_to_h(const uint4 w, uint4& lo4, uint4& hi4) {
    lo4.x = __byte_perm(w.x, 0x64646464u, 0x4140); lo4.y = __byte_perm(w.x, 0x64646464u, 0x4342);
    lo4.z = __byte_perm(w.y, 0x64646464u, 0x4140); lo4.w = __byte_perm(w.y, 0x64646464u, 0x4342);
    hi4.x = __byte_perm(w.z, 0x64646464u, 0x4140); hi4.y = __byte_perm(w.z, 0x64646464u, 0x4342);
    hi4.z = __byte_perm(w.w, 0x64646464u, 0x4140); hi4.w = __byte_perm(w.w, 0x64646464u, 0x4342);
}
// (1024 + byte) -> byte * scale, rounded once.  The fused form needs -1024 * scale inside the f16
// range; scales of 32 and more take the two-step form.
__device__ __forceinline__ void scale16(uint4& lo4, uint4& hi4, __half sc) {
    const uint32_t s2 = h2_bits(sc, sc);
    uint32_t* w0 = reinterpret_cast<uint32_t*>(&lo4);
    uint32_t* w1 = reinterpret_cast<uint32_t*>(&hi4);
    if (fabsf(__half2float(sc)) < 32.f) {
        const uint32_t c2 = hmul2_bits(s2, 0xE400E400u);   // -1024 * scale, exact
#pragma unroll
        for (int k = 0; k < 4; ++k) { w0[k] = hfma2_bits(w0[k], s2, c2); w1[k] = hfma2_bits(w1[k], s2, c2); }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) { w0[k] = hmul2_bits(hadd2_bits(w0[k], 0xE400E400u), s2); w1[k] = hmul2_bits(hadd2_bits(w1[k], 0xE400E400u), s2); }
    }
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
// (1024 + byte) -> (byte - 128) * scale, two values; the scales' two f16 pieces of each.  byte - 128 is exact, and the small piece's product is rounded far below the
// sum's own rounding: 2^-12 of a value in all, from the middle of the range.  With the scale rounded to one f16 (a multiply-add for three instructions) the result is
// 6.7e-4 off in all under f16 activations, 4.3e-4 so (u8 prompts 982 | 997 us, trees 291 | 293); integers as operands and both scales in the softmax leave
// 3.0e-4, the roundings of P and of the output, at 1137 | 335.
__device__ __forceinline__ uint32_t scale_two(uint32_t w, uint32_t high, uint32_t low) {
    const uint32_t b = hadd2_bits(w, 0xE480E480u);
    return hfma2_bits(b, high, hmul2_bits(b, low));
}
__device__ __forceinline__ void scale_eight(uint4& w4, uint2 sc) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&w4);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = scale_two(w[k], sc.x, sc.y);
}
// One arrival for the whole warp, after every lane's preceding writes.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}


__device__ __forceinline__ Item locate_item(const KernelArgs& a, int item, int G, int Hkv) {
    Item it;
    // q tiles in the plan's order (longest context first) when it made one, else in sequence order
    const int gq = a.plan->pitems_sorted ? __ldcg(a.pitem_order + item / Hkv) : item / Hkv;
    it.hk = item % Hkv;
    int lo = 0, hi = a.num_sequences;  // ptile_prefix[lo] <= gq < ptile_prefix[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(a.ptile_prefix + mid) <= gq) lo = mid; else hi = mid;
    }
    it.s = lo;
    const int p0 = __ldcg(a.ptile_prefix + lo), np = __ldcg(a.ptile_prefix + lo + 1) - p0;
    const int qt = np - 1 - (gq - p0);           // heavy (late) tiles first
    it.t0 = a.subsequence_begins[lo];
    it.n_new = a.subsequence_begins[lo + 1] - it.t0;
    it.past = a.past_lens[lo];
    it.table = a.block_indices + a.block_indices_begins[lo];
    it.row0 = qt * kPrefillItemRows;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r0 = it.row0 + x * kRows;
        if (r0 < it.n_new * G) {
            const int tok_hi = min(it.n_new - 1, (r0 + kRows - 1) / G);
            it.ctx_hi[x] = it.past + tok_hi + 1;
            it.nt[x] = (it.ctx_hi[x] + kKv - 1) / kKv;
        } else {
            it.ctx_hi[x] = 0;
            it.nt[x] = 0;
        }
    }
    it.ntiles = max(it.nt[0], it.nt[1]);
    return it;
}

// Walks CTA w's slice: the next piece of a list, false when there is none.
struct MaskWalk {
    MaskStart at, end;
    int Hkv, w;
    __device__ __forceinline__ MaskWalk(const KernelArgs& a, int cta) : Hkv(a.g.Hkv), w(cta) {
        const int4 s = __ldcg(reinterpret_cast<const int4*>(a.m.starts + cta)), e = __ldcg(reinterpret_cast<const int4*>(a.m.starts + cta + 1));
        at = MaskStart{s.x, s.y, s.z, 0};
        end = MaskStart{e.x, e.y, e.z, 0};
    }
    __device__ __forceinline__ bool next(const KernelArgs& a, int G, MaskedItem& it) {
        const bool last = at.q == end.q && at.hk == end.hk;
        if (at.q > end.q || (at.q == end.q && (at.hk > end.hk || (last && at.j >= end.j)))) return false;
        const int4* src = reinterpret_cast<const int4*>(a.m.items + at.q);
        const int4 x = __ldcg(src), y = __ldcg(src + 1);
        it.s = 0;
        it.hk = at.hk;
        it.t0 = x.x; it.n_new = x.y; it.past = x.z;
        it.table = a.block_indices + x.w;
        it.row0 = y.x; it.j0 = at.j;
        it.tree = y.z;
        const int end_j = last ? end.j : y.y, len = end_j - at.j;
        it.part = at.j > 0 ? 2 * w : end_j < y.y ? 2 * w + 1 : -1;
        const QTile q = q_tile(a.m, it.past, it.n_new, G, it.row0, it.tree);
        it.v = q.v;
        it.lo = q.lo;
        it.dup = q.cnt[1] == 0;
        it.ctx_hi[0] = q.ctx_hi[0];
        it.ctx_hi[1] = it.dup ? q.ctx_hi[0] : q.ctx_hi[1];
        it.nt[0] = it.dup ? (len + 1) / 2 : max(0, min(q.cnt[0], end_j) - at.j);
        it.nt[1] = it.dup ? len / 2 : max(0, min(q.cnt[1], end_j) - at.j);
        it.ntiles = it.dup ? len : max(it.nt[0], it.nt[1]);
        at.j = 0;
        if (++at.hk == Hkv) { at.hk = 0; ++at.q; }
        return true;
    }
};

#ifdef PA_PREFILL_PROF
// role (0, 1 softmax A, B; 2 converter; 3 mma; 4 loader; 5 second mma warp), event, tile 64..67 of CTA 0; 0: not met.  (In global
// memory: the 16-bit variants use all shared memory there is.)
constexpr int kTraceRoles = 6;
__device__ long long trace[kTraceRoles][8][4];
#endif

template <bool MK>
__device__ __forceinline__ auto make_walk(const KernelArgs& a) {
    if constexpr (MK) return MaskWalk(a, blockIdx.x);
    else return 0;
}

template <int BS, int CT, int D, bool MK>
__global__ void __launch_bounds__(kThreads, 1) prefill_tc_kernel(const __grid_constant__ KernelArgs a) {
    using Smem = PrefillSmem<BS, CT, D, MK>;
    using It = typename ItemOf<MK>::type;
    constexpr bool U8 = CT == PA_DTYPE_U8, BF = CT == PA_DTYPE_BF16;
    constexpr int kD = D, kNo = Smem::NO, kTmemP = 2 * kKv + 2 * kNo, NST = Smem::NST;
    // Masked: code that runs once an item stays in loops.  Straight through it is thousands of instructions that come from L2 every time: an epilogue
    // took 10 k cycles.
    constexpr int kRolled = MK ? 1 : 16;
    constexpr bool TwoMma = !U8 || MK;           // a warp issues the products of each half
    // tensor-memory columns of one half's P: f16, or bf16 high + low pieces.  (One bf16 piece leaves 2.3e-3 of the result in all where two leave the output's own
    // 1.7e-3; it costs a third of the products: masked ragged prompts 369 | 310 us, long trees 292 | 268.)
    constexpr int kPCols = BF ? kKv : kKv / 2;
    constexpr int kFmt = BF ? 1 : 0;
    static_assert(!U8 || NST == 2, "the converter and the loader of the u8 variant index two stages");
    static_assert(kTmemP + 2 * kPCols <= kTmemCols, "S, O and P of both halves fit the tensor memory");
    extern __shared__ uint8_t smem_raw_[];
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw_) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.g.Hq / a.g.Hkv;
    const int Hkv = a.g.Hkv;
    grid_wait();
    const int total_items = MK ? 0 : a.plan->total_ptiles * Hkv;
    const float qscale = (a.scale != 0.f ? a.scale : rsqrtf((float)kD)) * kLog2eP;

    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < NST; ++i) {
            if constexpr (U8) {
                mbar_init(&sm.raw_full[i], 1);
                mbar_init(&sm.raw_free[i], kConvWarps);
            }
            if constexpr (!U8 && MK) {
                mbar_init(&sm.k_full[i], 1);
                mbar_init(&sm.v_full[i], kConvWarps);
                mbar_init(&sm.v_land[i], 1);
            } else if constexpr (U8 && MK) {
                mbar_init(&sm.k_full[i], kConvWarps / 2);   // half of the converter's warps each
                mbar_init(&sm.v_full[i], kConvWarps / 2);
            } else {
                mbar_init(&sm.k_full[i], kConvWarps);
                mbar_init(&sm.v_full[i], kConvWarps);
            }
            mbar_init(&sm.k_free[i], TwoMma ? 2 : 1);   // one arrival per mma warp
            mbar_init(&sm.v_free[i], TwoMma ? 2 : 1);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            mbar_init(&sm.q_full[x], kRows / 32);
            mbar_init(&sm.s_full[x], 1);
            mbar_init(&sm.s_read[x], kRows / 32);
            mbar_init(&sm.p_full[x], kRows / 32);
            mbar_init(&sm.o_done[x], 1);
        }
#pragma unroll
        for (int i = 0; i < kItemSlots; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_free[i], kWarpMma + (TwoMma ? 2 : 1));
        }
        if constexpr (MK) {
            mbar_init(&sm.join_full, kRows / 32);
            mbar_init(&sm.join_free, kRows / 32);
        }
        mbar_fence_init();
        sm.abort = 0;
    }
    if constexpr (U8) {
        // rows 132..143 of V'^T stay zero for the whole kernel
        if (tid < NST * (kNo - kD - 4) * 8) {
            const int st = tid / ((kNo - kD - 4) * 8), i = tid % ((kNo - kD - 4) * 8);
            *reinterpret_cast<uint4*>(sm.vt[st] + (kD + 4) * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        }
    } else {
        // row 0 of the constant tile (16-byte units 0 and 8: its two halves along the tokens) is all ones
        if (!BF && tid < 32) {
            const uint32_t one2 = tid == 0 || tid == 8 ? 0x3C003C00u : 0u;
            *reinterpret_cast<uint4*>(sm.ones + tid * 16) = make_uint4(one2, one2, one2, one2);
        }
    }
    if (warp == 0) tc05::tmem_alloc(&sm.tmem_base, kTmemCols);
    tc05::fence_proxy_async_smem();
    tc05::fence_before_thread_sync();
    __syncthreads();
    tc05::fence_after_thread_sync();
    const uint32_t tmem = sm.tmem_base;

    [[maybe_unused]] uint32_t begun = 0, begun_v = 0;   // masked: tiles whose copies the loader has begun; whose values'
    // A wait that runs out raises sm.abort; every waiter polls the flag, so all roles unwind.
    // `cat` names the wait for the optional cycle accounting (-DPA_PREFILL_PROF).
#ifdef PA_PREFILL_PROF
    long long prof[5] = {0, 0, 0, 0, 0};
    const long long prof_begin = clock64();
    if (blockIdx.x == 0)
        for (int i = tid; i < kTraceRoles * 8 * 4; i += kThreads) (&trace[0][0][0])[i] = 0;
    __syncthreads();
#define PA_TRACE(role, ev, tile) do { if (lane == 0 && blockIdx.x == 0 && (tile) >= 64 && (tile) < 68) trace[role][ev][(tile) - 64] = clock64(); } while (0)
#else
#define PA_TRACE(role, ev, tile) do { } while (0)
#endif
    auto wait = [&](uint64_t* bar, uint32_t parity, int cat) -> bool {
#ifdef PA_PREFILL_PROF
        const long long w0 = clock64();
#endif
        bool ok = false;
        for (uint32_t i = 0; i < (1u << 22); ++i) {
            if (mbar_try_wait(bar, parity)) { ok = true; break; }
            if ((i & 255u) == 255u && sm.abort) return false;
        }
#ifdef PA_PREFILL_PROF
        prof[cat] += clock64() - w0;
#endif
        (void)cat;
        if (ok) return true;
        sm.abort = 1;
        atomicOr(a.status, PA_DEV_WAIT_TIMEOUT_PREFILL);
        return false;
    };
    auto wait_warp = [&](uint64_t* bar, uint32_t parity, int cat) -> bool { return __all_sync(0xffffffffu, wait(bar, parity, cat)) != 0; };
    // Work items come from a global counter: the loader draws them and publishes each through a
    // small ring, so that all roles of the CTA walk the same sequence.  -1 ends the sequence, -2
    // reports a wait that ran out.
    auto fetch_item = [&](uint32_t k, It& it) -> int {
        const int slot = k & (kItemSlots - 1);
        if (!wait_warp(&sm.item_full[slot], (k / kItemSlots) & 1, 0)) return -2;
        const int item = sm.item_ring[slot];
        if (item >= 0) it = sm.item_desc[slot];
        warp_arrive(&sm.item_free[slot]);
        return item;
    };

    // first context position of an item's j-th tile; whether any row of the item sees a position
    auto tile_pos = [&](const It& it, int j) -> int {   // (j counts the item's tiles, those of both halves)
        if constexpr (MK) return it.v.tile(it.j0 + j) * kKv;
        else return j * kKv;
    };
    auto seen = [&](const It& it, int ctx_hi, int pos) -> bool {
        if constexpr (MK) return pos < ctx_hi && (pos < a.m.sinks || pos >= it.lo);
        else return pos < ctx_hi;
    };

    // whether every token of a tile is seen by some row of the item
    [[maybe_unused]] auto whole_tile = [&](const It& it, int ctx_hi, int pos0) -> bool {
        if constexpr (MK) return pos0 + kKv <= ctx_hi && (pos0 >= it.lo || pos0 + kKv <= a.m.sinks);
        else return false;
    };

    if (warp >= kWarpMma) reg_dec<PA_TC_REG_MISC>();   // the fourth warpgroup: mma, loader, second mma; what is left over keeps it whole
    if (warp < kSoftmaxWarps) {
        // ======================= softmax + epilogue of half X ==========================================
        reg_inc<PA_TC_REG_SOFTMAX>();
        const int X = warp >> 2, r = tid & (kRows - 1);
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;   // this warp's TMEM lanes
        const uint32_t tmem_s = tmem + kKv * X + lane_base, tmem_o = tmem + 2 * kKv + kNo * X + lane_base;
        uint8_t* const sq = sm.q[X];
        const uint32_t tmem_p = tmem + kTmemP + kPCols * X + lane_base;
        uint32_t n = 0;   // tiles of this half so far, over all items
        uint32_t ik = 0;
        uint32_t joins = 0;        // masked: items whose results both halves hold, so far
        bool joins_open = false;   // half B: the last of them has not been read yet
        It it;
        // This thread's row of the item in work; the next item's is staged before this one's epilogue.
        struct Row {
            long long off;   // (token, q head) row of query / output
            int ctx;         // context it sees
            bool live;
            float qs;        // softmax scale: the kernel's, divided by the row's prescale
            int lo, tok;     // masked: begin of its window; its token's row of tree words, -1: no tree
        } row{0, 0, false, qscale, 0, -1};
        // The next item with rows in this half: 1, none left: 0, a wait ran out: -1
        auto next_item = [&]() -> int {
            for (;;) {
                const int item = fetch_item(ik, it);
                if (item == -2) return -1;
                if (item < 0) return 0;
                ++ik;
                if (it.nt[X] != 0) return 1;
            }
        };
        // Q -> swizzled A operand; the row's sum goes into the extra dims.  Every S of this half's previous item has
        // completed, so the tile is free.  16-bit rows: kD / 8 lanes take one row in 16-byte chunks, all loads of the warp's 32
        // rows in flight together (64 registers, free between items; cp.async where the row goes in as it is).  One thread per
        // row touched 32 lines with every load and, behind a branch on the type, had one load in flight: 10 k cycles an item.
        [[maybe_unused]] auto stage_q = [&]() {
            constexpr int CH = kD / 8, RP = 32 / CH;   // chunks of a row, rows per pass; CH passes
            const int flat = it.row0 + X * kRows + r;
            const int tok = flat / G, hq = it.hk * G + flat % G;
            row.live = tok < it.n_new;
            row.ctx = row.live ? it.past + tok + 1 : it.ctx_hi[X];
            row.off = ((long long)(it.t0 + (row.live ? tok : 0)) * a.g.Hq + hq);
            row.qs = qscale;
            const int wrow = r & ~31;                                  // the warp's first row
            const int own = row.live ? (int)row.off : -1;              // (rows fit 31 bits: 2^31 of them exceed the memory)
            const int ch = lane % CH, sub = lane / CH;
            uint8_t* const dst = sq + (ch / 8) * (kRows * 128);
            const uint4* const src = reinterpret_cast<const uint4*>(a.query) + ch;   // 16-bit rows of CH chunks
            if constexpr (BF) {   // bf16 activations only: the rows go in as they are
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int rr = RP * i + sub, o = __shfl_sync(0xffffffffu, own, rr);
                    cp_async16_zfill(dst + sw128(wrow + rr, ch & 7), src + (long long)max(o, 0) * CH, o >= 0 ? 16u : 0u);
                }
                cp_async_commit();
                cp_async_wait<0>();
            } else {
                // large queries (bf16 / f32 beyond the f16 range, or f16 rows whose sum would leave it): an exact power-of-two
                // prescale keeps the packed row and its sum inside the f16 range (the decode kernel does the same), and the
                // softmax scale of the row takes it back out
                auto prescale = [](float amax) {
                    float mul = 1.f;
                    if (amax > 256.f && amax < INFINITY) {   // 128 terms of at most 2^8 each keep the row sum below the f16 maximum too
                        int ex;
                        frexpf(amax, &ex);
                        mul = ldexpf(1.f, 8 - ex);
                    }
                    return mul;
                };
                auto sum8 = [](const uint4& w) {   // of the f16 values the tensor core will see
                    const __half2* h = reinterpret_cast<const __half2*>(&w);
                    float s4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s4[e] = __low2float(h[e]) + __high2float(h[e]);
                    return (s4[0] + s4[1]) + (s4[2] + s4[3]);
                };
                auto pack8 = [](const float (&v)[8], float mul) {
                    return make_uint4(pack_h2(v[0] * mul, v[1] * mul), pack_h2(v[2] * mul, v[3] * mul), pack_h2(v[4] * mul, v[5] * mul),
                                      pack_h2(v[6] * mul, v[7] * mul));
                };
                float qsum = 0.f;
                int sum_row = r;   // the row whose sum this thread ends up with
                if (a.g.act != PA_DTYPE_F32) {
                    uint4 raw[CH];
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        const int o = __shfl_sync(0xffffffffu, own, RP * i + sub);
                        raw[i] = o >= 0 ? src[(long long)o * CH] : make_uint4(0u, 0u, 0u, 0u);
                    }
                    const bool f16 = a.g.act == PA_DTYPE_F16;
                    auto values = [&](const uint4& q, float (&v)[8]) {
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                                 : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
                            v[2 * e] = f.x; v[2 * e + 1] = f.y;
                        }
                    };
                    // largest magnitude by bit pattern: both types order like their bits without the sign (NaN above all)
                    const uint32_t limit = f16 ? 0x5C00u : 0x4380u;   // 256
                    uint32_t top = 0u;
#pragma unroll
                    for (int i = 0; i < CH; ++i)
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu),
                                                     __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
                    const bool large = __any_sync(0xffffffffu, max(top & 0xffffu, top >> 16) > limit);
                    float sum[CH];
                    if (!large) {   // the usual case, straight through: nothing to scale
#pragma unroll
                        for (int i = 0; i < CH; ++i) {
                            uint4 w = raw[i];
                            if (!f16) {
                                float v[8];
                                values(raw[i], v);
                                w = pack8(v, 1.f);
                            }
                            *reinterpret_cast<uint4*>(dst + sw128(wrow + RP * i + sub, ch & 7)) = w;
                            if constexpr (U8) sum[i] = sum8(w);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < CH; ++i) {
                            float v[8];
                            values(raw[i], v);
                            float m = 0.f;
#pragma unroll
                            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
#pragma unroll
                            for (int o = CH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                            const float mul = prescale(m);
                            const float mine = __shfl_sync(0xffffffffu, mul, (lane % RP) * CH);   // row RP i + lane % RP
                            if (lane / RP == i) row.qs = qscale / mine;
                            const uint4 w = pack8(v, mul);
                            *reinterpret_cast<uint4*>(dst + sw128(wrow + RP * i + sub, ch & 7)) = w;
                            if constexpr (U8) sum[i] = sum8(w);
                        }
                    }
                    if constexpr (U8) {
                        // sums over the CH lanes of every row at once: each step halves the rows a lane carries, and lane
                        // (sub, ch) is left with row RP ch + sub
#pragma unroll
                        for (int o = CH / 2; o > 0; o >>= 1) {
                            const bool hi = (ch & o) != 0;
#pragma unroll
                            for (int k = 0; k < o; ++k) {
                                const float give = hi ? sum[k] : sum[k + o], keep = hi ? sum[k + o] : sum[k];
                                sum[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                            }
                        }
                        qsum = sum[0];
                        sum_row = wrow + RP * ch + sub;
                    }
                } else {
                    float amax = 0.f;
#pragma unroll 4
                    for (int c = 0; c < CH; ++c) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = 0.f;
                        if (row.live) load_act_vec<8>(a.query, row.off * kD + 8 * c, a.g.act, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
                    }
                    const float mul = prescale(amax);
                    row.qs = qscale / mul;
#pragma unroll 4
                    for (int c = 0; c < CH; ++c) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = 0.f;
                        if (row.live) load_act_vec<8>(a.query, row.off * kD + 8 * c, a.g.act, v);
                        const uint4 w = pack8(v, mul);
                        *reinterpret_cast<uint4*>(sq + (c / 8) * (kRows * 128) + sw128(r, c % 8)) = w;
                        if constexpr (U8) qsum += sum8(w);
                    }
                }
                if constexpr (U8) {
                    const __half qh = f2h(qsum), ql = f2h(qsum - __half2float(qh));
                    const __half zero = __ushort_as_half(0);
                    *reinterpret_cast<uint4*>(sm.qx[X] + plain16(sum_row, 0)) = make_uint4(h2_bits(qh, qh), h2_bits(qh, ql), h2_bits(ql, zero), 0u);
                    *reinterpret_cast<uint4*>(sm.qx[X] + plain16(sum_row, 1)) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            tc05::fence_proxy_async_smem();
            warp_arrive(&sm.q_full[X]);
        };
        // Masked, 16-bit activations: the rows go into the operand tile as they are, asynchronously (stage_begin), and are looked through and converted
        // where they lie (stage_end), in short loops; between the two lies the epilogue of the item before.
        [[maybe_unused]] auto place_row = [&] {
            int flat = it.row0 + X * kRows + r;
            if constexpr (MK) flat -= it.dup ? X * kRows : 0;
            const int tok = flat / G, hq = it.hk * G + flat % G;
            row.live = tok < it.n_new;
            row.off = (long long)(it.t0 + (row.live ? tok : 0)) * a.g.Hq + hq;
            row.qs = qscale;
            if constexpr (MK) {
                row.tok = -1;
                row.ctx = 0x7fffffff; row.lo = 0;   // (a row that is none sees zeros)
                if (row.live && it.tree) {
                    row.tok = it.t0 + tok;
                    row.ctx = it.past;
                    row.lo = window_lo(a.m, it.past + __ldcg(a.m.tree_depth + row.tok) + 1);
                } else if (row.live) {
                    row.ctx = it.past + tok + 1;
                    row.lo = window_lo(a.m, row.ctx);
                }
            }
        };
        constexpr int CH = kD / 8, RP = 32 / CH;   // 16-byte chunks of a row, rows of a warp side by side
        [[maybe_unused]] auto stage_begin = [&] {
            place_row();
            if (a.g.act == PA_DTYPE_F32) return;
            const int own = row.live ? (int)row.off : -1, ch = lane % CH, sub = lane / CH;
            uint8_t* const dst = sq + (ch / 8) * (kRows * 128);
            const uint4* const src = reinterpret_cast<const uint4*>(a.query) + ch;
#pragma unroll 4
            for (int i = 0; i < CH; ++i) {
                const int o = __shfl_sync(0xffffffffu, own, RP * i + sub);
                cp_async16_zfill(dst + sw128((r & ~31) + RP * i + sub, ch & 7), src + (long long)max(o, 0) * CH, o >= 0 ? 16u : 0u);
            }
            cp_async_commit();
        };
        [[maybe_unused]] auto stage_end = [&] {
            const int ch = lane % CH, sub = lane / CH, wrow = r & ~31;
            uint8_t* const dst = sq + (ch / 8) * (kRows * 128);
            float qsum = 0.f;
            // the row whose sum this thread ends up with: of turn ch % (CH / 4), the one that its upper two bits choose
            int sum_row = wrow + RP * (4 * (ch & (CH / 4 - 1)) + (ch >> (CH == 16 ? 2 : 1))) + sub;
            auto sum8 = [](const uint4& w) {      // of the f16 values the tensor core will see
                const __half2* h = reinterpret_cast<const __half2*>(&w);
                float s4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) s4[e] = __low2float(h[e]) + __high2float(h[e]);
                return (s4[0] + s4[1]) + (s4[2] + s4[3]);
            };
            auto pack8 = [](const float (&v)[8], float mul) {
                return make_uint4(pack_h2(v[0] * mul, v[1] * mul), pack_h2(v[2] * mul, v[3] * mul), pack_h2(v[4] * mul, v[5] * mul), pack_h2(v[6] * mul, v[7] * mul));
            };
            // large queries: an exact power of two that keeps row and sum inside the f16 range, taken back out by the row's softmax scale (as stage_q says)
            auto prescale = [](float amax) {
                float mul = 1.f;
                if (amax > 256.f && amax < INFINITY) {
                    int ex;
                    frexpf(amax, &ex);
                    mul = ldexpf(1.f, 8 - ex);
                }
                return mul;
            };
            if (a.g.act != PA_DTYPE_F32) {
                cp_async_wait<0>();
                __syncwarp();
                if constexpr (!BF) {
                    const bool f16 = a.g.act == PA_DTYPE_F16;
                    auto values = [&](const uint4& q, float (&v)[8]) {
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[e]))
                                                 : make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
                            v[2 * e] = f.x; v[2 * e + 1] = f.y;
                        }
                    };
                    const uint32_t limit = f16 ? 0x5C00u : 0x4380u;   // 256, by bit pattern
                    uint32_t top = 0u;
#pragma unroll 4
                    for (int i = 0; i < CH; ++i) {
                        const uint4 w = *reinterpret_cast<const uint4*>(dst + sw128(wrow + RP * i + sub, ch & 7));
                        top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
                    }
                    const bool large = __any_sync(0xffffffffu, max(top & 0xffffu, top >> 16) > limit);
                    if (U8 || !f16 || large) {
                        // four rows a turn: converted where they lie, and their sums over the CH lanes of a row together: two steps that halve the rows a
                        // lane carries, then those over what is left of the lanes (one row after the other it was four steps each, 5 - 9 k cycles)
                        static_assert(CH % 4 == 0, "whole turns");
#pragma unroll 1
                        for (int b = 0; b < CH / 4; ++b) {
                            uint4* at[4];
                            uint4 w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                at[i] = reinterpret_cast<uint4*>(dst + sw128(wrow + RP * (4 * b + i) + sub, ch & 7));
                                w[i] = *at[i];
                            }
                            if (!f16 || large) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    float v[8], mul = 1.f;
                                    values(w[i], v);
                                    if (large) {
                                        float m = 0.f;
#pragma unroll
                                        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
#pragma unroll
                                        for (int o = CH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                                        mul = prescale(m);
                                        const float mine = __shfl_sync(0xffffffffu, mul, (lane % RP) * CH);   // row RP (4 b + i) + lane % RP
                                        if (lane / RP == 4 * b + i) row.qs = qscale / mine;
                                    }
                                    w[i] = pack8(v, mul);
                                    *at[i] = w[i];
                                }
                            }
                            if constexpr (U8) {
                                float t[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) t[i] = sum8(w[i]);
                                const bool hi = (ch & (CH / 2)) != 0, hi2 = (ch & (CH / 4)) != 0;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const float give = hi ? t[i] : t[i + 2], keep = hi ? t[i + 2] : t[i];
                                    t[i] = keep + __shfl_xor_sync(0xffffffffu, give, CH / 2);
                                }
                                float s = (hi2 ? t[1] : t[0]) + __shfl_xor_sync(0xffffffffu, hi2 ? t[0] : t[1], CH / 4);
#pragma unroll
                                for (int o = CH / 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                                if ((ch & (CH / 4 - 1)) == b) qsum = s;
                            }
                        }
                    }
                }
            } else {
                sum_row = r;
                float amax = 0.f;
#pragma unroll 4
                for (int c = 0; c < CH; ++c) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.f;
                    if (row.live) load_act_vec<8>(a.query, row.off * kD + 8 * c, a.g.act, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
                }
                const float mul = prescale(amax);
                row.qs = qscale / mul;
#pragma unroll 4
                for (int c = 0; c < CH; ++c) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.f;
                    if (row.live) load_act_vec<8>(a.query, row.off * kD + 8 * c, a.g.act, v);
                    const uint4 w = pack8(v, mul);
                    *reinterpret_cast<uint4*>(sq + (c / 8) * (kRows * 128) + sw128(r, c % 8)) = w;
                    if constexpr (U8) qsum += sum8(w);
                }
            }
            if constexpr (U8) {
                const __half qh = f2h(qsum), ql = f2h(qsum - __half2float(qh));
                const __half zero = __ushort_as_half(0);
                *reinterpret_cast<uint4*>(sm.qx[X] + plain16(sum_row, 0)) = make_uint4(h2_bits(qh, qh), h2_bits(qh, ql), h2_bits(ql, zero), 0u);
                *reinterpret_cast<uint4*>(sm.qx[X] + plain16(sum_row, 1)) = make_uint4(0u, 0u, 0u, 0u);
            }
            tc05::fence_proxy_async_smem();
            warp_arrive(&sm.q_full[X]);
        };
        int have = next_item();
        if (have < 0) goto done;
        if (have) {
            if constexpr (MK) {
                stage_begin();
                stage_end();
            } else {
                stage_q();
            }
        }
        while (have) {
            const int nt = it.nt[X], my_ctx = row.ctx;
            const float qs = row.qs;
            int my_lo = 0, my_tok = -1;
            if constexpr (MK) { my_lo = row.lo; my_tok = row.tok; }

            float m_run = -INFINITY;   // running maximum of q.k' (before the softmax scale)
            float l_own = 0.f;         // bf16 variant: the row's own sum of probabilities
            for (int j = 0; j < nt; ++j, ++n) {
                int col0;
                if constexpr (MK) col0 = tile_pos(it, it.dup ? 2 * j + X : j);
                else col0 = tile_pos(it, j);
                if (!wait_warp(&sm.s_full[X], n & 1, 0)) goto done;
                if ((warp & 3) == 0) PA_TRACE(X, 0, n);
                tc05::fence_after_thread_sync();
                float sv[kKv];   // q.k' in units of 1 / qs
                {
                    uint32_t s0[32], s1[32];
                    tc05::ld_32x32b_x32(tmem_s, s0);
                    tc05::ld_32x32b_x32(tmem_s + 32, s1);
                    tc05::wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) { sv[c] = __uint_as_float(s0[c]); sv[32 + c] = __uint_as_float(s1[c]); }
                }
                if constexpr (TwoMma) {
                    tc05::fence_before_thread_sync();
                    warp_arrive(&sm.s_read[X]);
                }
                if ((warp & 3) == 0) PA_TRACE(X, 1, n);
                if constexpr (MK) {            // a tile that this row does not see as a whole
                    if (col0 + kKv > my_ctx || (col0 < my_lo && col0 + kKv > a.m.sinks)) {
                        uint64_t w = causal_bits(col0, my_ctx, my_lo, a.m.sinks);
                        if (my_tok >= 0 && col0 + kKv > it.past) w |= tree_bits64(a.m.tree_words + (long long)my_tok * kTreeWords, col0 - it.past);
                        const uint32_t w0 = (uint32_t)w, w1 = (uint32_t)(w >> 32);
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            sv[c] = (w0 >> c) & 1u ? sv[c] : -INFINITY;
                            sv[32 + c] = (w1 >> c) & 1u ? sv[32 + c] : -INFINITY;
                        }
                    }
                } else if (col0 + kKv > my_ctx) {     // diagonal tile: hide what this row cannot see
                    const int nvis = my_ctx - col0;   // may be <= 0
#pragma unroll
                    for (int c = 0; c < kKv; ++c) sv[c] = c < nvis ? sv[c] : -INFINITY;
                }
                float mx = -INFINITY;
                if constexpr (MK) {   // four chains: one of 32 links is as long as the exponentials
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < kKv; c += 2) m4[(c >> 1) & 3] = max3(m4[(c >> 1) & 3], sv[c], sv[c + 1]);
                    mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
                } else {
#pragma unroll
                    for (int c = 0; c < kKv; c += 2) mx = max3(mx, sv[c], sv[c + 1]);
                }
                float alpha = 1.f;
                bool rescale = false;
                if (j == 0) {
                    m_run = mx;      // finite: column 0 of tile 0 is visible to every row (masked: of a first tile a row may see nothing)
                } else {
                    const bool grow = (mx - m_run) * qs > kLazy;
                    rescale = __any_sync(0xffffffffu, grow);
                    if (grow) { alpha = ex2((m_run - mx) * qs); m_run = mx; }
                }
                if constexpr (BF) l_own *= alpha;
                // P = 2^(qs * (s - m)) in f16 pairs: the exponent is rounded to f16 first, which costs
                // at most 2^-12 of the exponent's magnitude in relative error of p
                [[maybe_unused]] float2 l2 = make_float2(0.f, 0.f);
                const float mq = MK && m_run == -INFINITY ? 0.f : m_run * qs;   // (nothing seen yet: every p is 0)
                uint32_t pw[kKv / 2];
                uint32_t pl[BF ? kKv / 2 : 1];   // bf16 variant: the low pieces, p = high + low up to 2^-17 p
#pragma unroll
                for (int c = 0; c < kKv; c += 2) {
                    // the packed f16 exponential is good to 2^-9.9 relative: inside the u8 cache's error bound, not inside the
                    // f16 cache's, whose P goes through the f32 exponential and is rounded once
                    if constexpr (MK) {   // of every cache, as for f16, with the scaling and the row's sum two at a time (u8 prompts 1027 us packed, 964 so)
                        const float2 x = fma_pair(sv[c], sv[c + 1], qs, -mq);
                        const float2 p = make_float2(ex2(x.x), ex2(x.y));
                        if constexpr (BF) {
                            l2 = add_pair(l2, p);
                            const uint32_t hi = pack_bf2(p.x, p.y);
                            pw[c >> 1] = hi;
                            pl[c >> 1] = pack_bf2(p.x - __uint_as_float(hi << 16), p.y - __uint_as_float(hi & 0xffff0000u));
                        } else {
                            pw[c >> 1] = pack_h2(p.x, p.y);
                        }
                    } else if constexpr (U8) {
                        pw[c >> 1] = ex2_h2(pack_h2(fmaf(sv[c], qs, -mq), fmaf(sv[c + 1], qs, -mq)));
                    } else if constexpr (BF) {
                        const float p0 = ex2(fmaf(sv[c], qs, -mq)), p1 = ex2(fmaf(sv[c + 1], qs, -mq));
                        l_own += p0 + p1;
                        const uint32_t hi = pack_bf2(p0, p1);
                        pw[c >> 1] = hi;
                        pl[c >> 1] = pack_bf2(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u));
                    } else {
                        pw[c >> 1] = pack_h2(ex2(fmaf(sv[c], qs, -mq)), ex2(fmaf(sv[c + 1], qs, -mq)));
                    }
                }
                if constexpr (MK && BF) l_own += l2.x + l2.y;
                // P.V of the previous tile of this half still reads the P tile and writes O
                if ((warp & 3) == 0) PA_TRACE(X, 2, n);
                if (n > 0) {
                    if (!wait_warp(&sm.o_done[X], (n - 1) & 1, 1)) goto done;
                    tc05::fence_after_thread_sync();
                }
                if constexpr (MK) {   // half A may still be reading the last item's results of half B
                    if (joins_open) {
                        if (!wait_warp(&sm.join_free, (joins - 1) & 1, 1)) goto done;
                        joins_open = false;
                    }
                }
                if ((warp & 3) == 0) PA_TRACE(X, 3, n);
                if (rescale) {
#pragma unroll kRolled
                    for (int q4 = 0; q4 < kD / 32; ++q4) {
                        uint32_t t[32];
                        tc05::ld_32x32b_x32(tmem_o + 32 * q4, t);
                        tc05::wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) t[c] = __float_as_uint(__uint_as_float(t[c]) * alpha);
                        tc05::st_32x32b_x32(tmem_o + 32 * q4, t);
                    }
                    if constexpr (!BF) {
                        uint32_t t[16];
                        tc05::ld_32x32b_x16(tmem_o + kD, t);
                        tc05::wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; ++c) t[c] = __float_as_uint(__uint_as_float(t[c]) * alpha);
                        tc05::st_32x32b_x16(tmem_o + kD, t);
                    }
                    tc05::wait_st();
                }
                tc05::st_32x32b_x32(tmem_p, pw);   // row r of the A operand: lane r, two tokens per column
                if constexpr (BF) tc05::st_32x32b_x32(tmem_p + kKv / 2, pl);
                tc05::wait_st();
                tc05::fence_before_thread_sync();
                warp_arrive(&sm.p_full[X]);
                if ((warp & 3) == 0) PA_TRACE(X, 4, n);
            }
            // ---- the next item's rows, so that its first logits are computed beside this item's last P.V and epilogue (its
            // first P, which starts a new O, comes after) ---------------------------------------------------
            const Row cur = row;
            int part = -1;
            bool dup = false;
            if constexpr (MK) { part = it.part; dup = it.dup && it.nt[1] > 0; }
            have = next_item();
            if (have < 0) goto done;
            if (have) {
                if constexpr (MK) stage_begin();
                else stage_q();
            }
            // ---- epilogue: out = (O - z) / l; z = the three zero-point columns, l = the all-ones column (u8 cache);
            // the f16 cache has no z and its l is the first column of the 16-column product
            if (!wait_warp(&sm.o_done[X], (n - 1) & 1, 2)) goto done;
            tc05::fence_after_thread_sync();
            // masked: both halves have worked on these rows; half A takes fa of its own results and fb of half B's, which lie in the same lanes
            float fa = 1.f, fb = 0.f, zb = 0.f, lb = 0.f;
            if constexpr (MK) {
                if (dup) {
                    ++joins;
                    if (X == 1) {
                        reinterpret_cast<float2*>(sm.out_stage[warp])[lane] = make_float2(m_run * cur.qs, l_own);
                        tc05::fence_before_thread_sync();
                        warp_arrive(&sm.join_full);
                        joins_open = true;
                        if (have) stage_end();
                        continue;
                    }
                    if (!wait_warp(&sm.join_full, (joins - 1) & 1, 2)) goto done;
                    tc05::fence_after_thread_sync();
                    const float2 other = reinterpret_cast<const float2*>(sm.out_stage[warp + 4])[lane];
                    const float ma = m_run * cur.qs, top = fmaxf(ma, other.x);
                    fa = ma == -INFINITY ? 0.f : ex2(ma - top);
                    fb = other.x == -INFINITY ? 0.f : ex2(other.x - top);
                    m_run = top / cur.qs;
                    lb = other.y;
                    if constexpr (!BF) {
                        uint32_t zr[16];
                        tc05::ld_32x32b_x16(tmem_o + kNo + kD, zr);
                        tc05::wait_ld();
                        if constexpr (U8) zb = __uint_as_float(zr[0]) + __uint_as_float(zr[1]) + __uint_as_float(zr[2]);
                        lb = __uint_as_float(zr[U8 ? 3 : 0]);
                    }
                }
            }
            {
                float z = 0.f, l_run = l_own;
                if constexpr (!BF) {
                    uint32_t zr[16];
                    tc05::ld_32x32b_x16(tmem_o + kD, zr);
                    tc05::wait_ld();
                    if constexpr (U8) z = __uint_as_float(zr[0]) + __uint_as_float(zr[1]) + __uint_as_float(zr[2]);
                    l_run = __uint_as_float(zr[U8 ? 3 : 0]);
                }
                if constexpr (MK) {
                    if (dup) { z = fa * z + fb * zb; l_run = fa * l_run + fb * lb; }
                }
                // columns of the row's results, of both halves where both have some
                auto results = [&](int col, uint32_t (&t)[32]) {
                    tc05::ld_32x32b_x32(tmem_o + col, t);
                    tc05::wait_ld();
                    if constexpr (MK) {
                        if (dup) {
                            uint32_t u[32];
                            tc05::ld_32x32b_x32(tmem_o + kNo + col, u);
                            tc05::wait_ld();
#pragma unroll
                            for (int c = 0; c < 32; ++c) t[c] = __float_as_uint(fa * __uint_as_float(t[c]) + fb * __uint_as_float(u[c]));
                        }
                    }
                };
                const bool whole = !MK || part < 0;   // else a piece: unnormalised, to the scratch
                const float inv = whole ? 1.f / l_run : 1.f;
                // 128 bytes of every row at a time, turned around in shared memory so that eight lanes store one row's piece (a
                // thread storing its own row touched 32 lines with every store: 7 k cycles an item)
                uint8_t* const stg = sm.out_stage[warp];
                const int own = cur.live ? (whole ? (int)cur.off : X * kRows + r) : -1;
                uint8_t* const dst = whole ? (uint8_t*)a.output : (uint8_t*)(a.m.part_o + (long long)part * kPrefillItemRows * kD);
                const int c8 = lane & 7;
                [[maybe_unused]] float odd = 0.f;   // masked: not-a-number once a result is not finite, which may come from what the row does not see
                auto put = [&](int c, const uint4& w) { *reinterpret_cast<uint4*>(stg + lane * 128 + ((c ^ (lane & 7)) << 4)) = w; };
                auto send = [&](int piece, int row_bytes) {   // the piece of every row of the warp
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int rr = 4 * i + (lane >> 3), o = __shfl_sync(0xffffffffu, own, rr);
                        const uint4 w = *reinterpret_cast<const uint4*>(stg + rr * 128 + ((c8 ^ (rr & 7)) << 4));
                        if (o >= 0) *reinterpret_cast<uint4*>(dst + (long long)o * row_bytes + 128 * piece + 16 * c8) = w;
                    }
                    __syncwarp();
                };
                if (a.g.act == PA_DTYPE_F32 || !whole) {
#pragma unroll kRolled
                    for (int q4 = 0; q4 < kD / 32; ++q4) {
                        uint32_t t[32];
                        results(32 * q4, t);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (MK) {
                                    const float v = fmaf(__uint_as_float(t[4 * c + e]), inv, -z * inv);
                                    odd = fmaf(v, 0.f, odd);
                                    w[e] = __float_as_uint(v);
                                } else {
                                    w[e] = __float_as_uint((__uint_as_float(t[4 * c + e]) - z) * inv);
                                }
                            }
                            put(c, make_uint4(w[0], w[1], w[2], w[3]));
                        }
                        send(q4, kD * 4);
                    }
                } else {
                    const bool f16 = a.g.act == PA_DTYPE_F16;
#pragma unroll kRolled
                    for (int q = 0; q < kD / 64; ++q) {
#pragma unroll kRolled
                        for (int h = 0; h < 2; ++h) {
                            uint32_t t[32];
                            results(64 * q + 32 * h, t);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float v0, v1;
                                    if constexpr (MK) {
                                        v0 = fmaf(__uint_as_float(t[8 * c + 2 * e]), inv, -z * inv);
                                        v1 = fmaf(__uint_as_float(t[8 * c + 2 * e + 1]), inv, -z * inv);
                                        odd = fmaf(v0, 0.f, odd);
                                        odd = fmaf(v1, 0.f, odd);
                                    } else {
                                        v0 = (__uint_as_float(t[8 * c + 2 * e]) - z) * inv;
                                        v1 = (__uint_as_float(t[8 * c + 2 * e + 1]) - z) * inv;
                                    }
                                    w[e] = f16 ? pack_h2(v0, v1) : pack_bf2(v0, v1);
                                }
                                put(4 * h + c, make_uint4(w[0], w[1], w[2], w[3]));
                            }
                        }
                        send(q, kD * 2);
                    }
                }
                if (MK && whole && cur.live && odd != 0.f) a.m.redo[atomicAdd(&a.plan->total_redo, 1)] = (int)cur.off;
                if (MK && !whole) {
                    if (cur.live) a.m.part_ml[(long long)part * kPrefillItemRows + X * kRows + r] = make_float2(m_run * cur.qs, l_run);
                } else if (cur.live && a.lse) {
                    a.lse[cur.off] = (m_run * cur.qs + log2f(l_run)) * kLn2P;
                }
            }
            tc05::fence_before_thread_sync();
            if constexpr (MK) {
                if (dup) warp_arrive(&sm.join_free);
                if (have) stage_end();
            }
        }
    } else if (warp < kWarpMma) {
        // ======================= converter: raw records -> f16 operand tiles =============================
        reg_dec<PA_TC_REG_CONV>();
        const int ctid = tid - kSoftmaxWarps * 32, cwarp = warp - kSoftmaxWarps;
        if constexpr (U8 && MK) {
            // Masked: two warps for the keys and two for the values, so that neither's waits and fences hold up the other's (one behind the other, keys and
            // values took 2900 cycles of a tile's 3600).  All loads of a batch of units come first.
            const bool values = cwarp >= kConvWarps / 2;
            const int gt = ctid & 63;
            constexpr int NB = 4;   // units of a batch
            uint32_t t = 0;   // tiles so far, over all items
            for (uint32_t ik = 0;; ++ik) {
                It it;
                const int item = fetch_item(ik, it);
                if (item == -2) goto done;
                if (item < 0) break;
                const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
                for (int j = 0; j < it.ntiles; ++j, ++t) {
                    const int st = t & 1, pos0 = tile_pos(it, j);
                    const uint32_t use = t >> 1;
                    const uint8_t* const raw = values ? sm.raw_v[st] : sm.raw_k[st];
                    if (!wait_warp(&sm.raw_full[st], use & 1, 0)) goto done;
                    // every warp has the scales of all tokens (so that none waits for another); this thread sees to the zero-point of token gt
                    uint2* const tok = sm.tok_scale[cwarp];
                    float z = 0.f;   // of token gt: (byte - zp) * scale = operand - z
                    bool ok = false;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int token = 32 * h + lane;
                        const bool live = seen(it, ctx_hi, pos0 + token);
                        const float* const par = reinterpret_cast<const float*>(raw + (token / BS) * Smem::RSTRIDE + BS * kD) + token % BS;
                        const float scale = live ? par[0] : 0.f;   // (a token that no row sees becomes zeros)
                        __half high = f2h(scale);
                        const __half low = f2h(scale - __half2float(high));
                        // -128 * scale leaves the f16 range just behind 511.  Of a key that would be a logit of -infinity, which hides the token as a mask does: not a
                        // number instead, so that the rows that see it are computed again in 32 bits (masked_row).
                        if (!(fabsf(scale) < 511.f)) high = __ushort_as_half(0x7FFFu);
                        tok[token] = make_uint2(h2_bits(high, high), h2_bits(low, low));
                        if (token == gt) {
                            ok = live;
                            z = live ? scale * (par[BS] - 128.f) : 0.f;
                        }
                    }
                    const __half zero = __ushort_as_half(0);
                    __half zh, zm, zl;
                    split3(values ? z : -z, zh, zm, zl);
                    __syncwarp();
                    if (!values) {
                        if (use > 0 && !wait_warp(&sm.k_free[st], (use - 1) & 1, 1)) goto done;
                        // K' = (byte - 128) * k scale: unit = 16 dims of one token
                        *reinterpret_cast<uint4*>(sm.kx[st] + plain16(gt, 0)) = make_uint4(h2_bits(zh, zm), h2_bits(zl, zh), h2_bits(zm, zero), 0u);
                        *reinterpret_cast<uint4*>(sm.kx[st] + plain16(gt, 1)) = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
                        for (int u0 = gt; u0 < kKv * (kD / 16); u0 += 64 * NB) {
                            uint4 lo4[NB], hi4[NB];
                            uint2 sc[NB];
#pragma unroll
                            for (int i = 0; i < NB; ++i) {
                                const int u = u0 + 64 * i, token = u / (kD / 16), seg = u % (kD / 16);
                                sc[i] = tok[token];
                                bytes16_to_h(*reinterpret_cast<const uint4*>(raw + (token / BS) * Smem::RSTRIDE + (token % BS) * kD + 16 * seg), lo4[i], hi4[i]);
                            }
#pragma unroll
                            for (int i = 0; i < NB; ++i) {
                                const int u = u0 + 64 * i, token = u / (kD / 16), seg = u % (kD / 16);
                                scale_eight(lo4[i], sc[i]);
                                scale_eight(hi4[i], sc[i]);
                                uint8_t* atom = sm.k[st] + (seg >> 2) * (kKv * 128);
                                *reinterpret_cast<uint4*>(atom + sw128(token, (2 * seg) & 7)) = lo4[i];
                                *reinterpret_cast<uint4*>(atom + sw128(token, (2 * seg + 1) & 7)) = hi4[i];
                            }
                        }
                        tc05::fence_proxy_async_smem();
                        warp_arrive(&sm.k_full[st]);
                    } else {
                        if (use > 0 && !wait_warp(&sm.v_free[st], (use - 1) & 1, 2)) goto done;
                        // V'^T = (byte - 128) * v scale: unit = 16 tokens of one dim
                        const int tg = gt & 3;
                        uint2 tab[8];   // of two tokens: their scales' two pieces
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint4 two = *reinterpret_cast<const uint4*>(&tok[16 * tg + 2 * k]);
                            tab[k] = make_uint2(__byte_perm(two.x, two.z, 0x5410), __byte_perm(two.y, two.w, 0x5410));
                        }
                        constexpr int UPR = BS / 16;   // 16-token units per record
                        const uint8_t* const col = raw + (tg / UPR) * Smem::RSTRIDE + 16 * (tg % UPR);
#pragma unroll 1
                        for (int d0 = gt >> 2; d0 < kD; d0 += 16 * NB) {
                            uint4 lo4[NB], hi4[NB];
#pragma unroll
                            for (int i = 0; i < NB; ++i) bytes16_to_h(*reinterpret_cast<const uint4*>(col + (d0 + 16 * i) * BS), lo4[i], hi4[i]);
#pragma unroll
                            for (int i = 0; i < NB; ++i) {
                                const int d = d0 + 16 * i;
                                uint32_t w[8] = {lo4[i].x, lo4[i].y, lo4[i].z, lo4[i].w, hi4[i].x, hi4[i].y, hi4[i].z, hi4[i].w};
#pragma unroll
                                for (int k = 0; k < 8; ++k) w[k] = scale_two(w[k], tab[k].x, tab[k].y);
                                *reinterpret_cast<uint4*>(sm.vt[st] + sw128(d, 2 * tg)) = make_uint4(w[0], w[1], w[2], w[3]);
                                *reinterpret_cast<uint4*>(sm.vt[st] + sw128(d, 2 * tg + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        }
                        const uint32_t off = (gt & 7) * 2;
                        uint8_t* vt = sm.vt[st];
                        *reinterpret_cast<__half*>(vt + sw128(kD + 0, gt >> 3) + off) = zh;
                        *reinterpret_cast<__half*>(vt + sw128(kD + 1, gt >> 3) + off) = zm;
                        *reinterpret_cast<__half*>(vt + sw128(kD + 2, gt >> 3) + off) = zl;
                        *reinterpret_cast<__half*>(vt + sw128(kD + 3, gt >> 3) + off) = __ushort_as_half(ok ? (unsigned short)0x3C00u : (unsigned short)0u);
                        tc05::fence_proxy_async_smem();
                        warp_arrive(&sm.v_full[st]);
                    }
                    warp_arrive(&sm.raw_free[st]);   // (and the scales have been read)
                }
            }
        } else if constexpr (U8) {
        uint32_t t = 0;   // tiles so far, over all items
        for (uint32_t ik = 0;; ++ik) {
            It it;
            const int item = fetch_item(ik, it);
            if (item == -2) goto done;
            if (item < 0) break;
            const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
            for (int j = 0; j < it.ntiles; ++j, ++t) {
                const int st = t & 1;
                const uint32_t use = t >> 1;
                const int pos0 = tile_pos(it, j);
                const uint8_t* raw_k = sm.raw_k[st];
                const uint8_t* raw_v = sm.raw_v[st];
                if (!wait_warp(&sm.raw_full[st], use & 1, 0)) goto done;
                if (cwarp == 0) PA_TRACE(2, 0, t);
                if (use > 0 && !wait_warp(&sm.k_free[st], (use - 1) & 1, 1)) goto done;
                if (cwarp == 0) PA_TRACE(2, 1, t);
                // K' = byte * f16(k scale): unit u = 16 dims of one token
#pragma unroll
                for (int i = 0; i < kD / 32; ++i) {
                    const int u = ctid + 128 * i;
                    const int token = u / (kD / 16), seg = u % (kD / 16);
                    uint4 lo4 = make_uint4(0u, 0u, 0u, 0u), hi4 = lo4;
                    if (seen(it, ctx_hi, pos0 + token)) {
                        const uint8_t* rec = raw_k + (token / BS) * Smem::RSTRIDE;
                        const __half ksh = f2h(*reinterpret_cast<const float*>(rec + BS * kD + 4 * (token % BS)));
                        bytes16_to_h(*reinterpret_cast<const uint4*>(rec + (token % BS) * kD + 16 * seg), lo4, hi4);
                        scale16(lo4, hi4, ksh);
                    }
                    uint8_t* atom = sm.k[st] + (seg >> 2) * (kKv * 128);
                    *reinterpret_cast<uint4*>(atom + sw128(token, (2 * seg) & 7)) = lo4;
                    *reinterpret_cast<uint4*>(atom + sw128(token, (2 * seg + 1) & 7)) = hi4;
                }
                if (ctid < kKv) {
                    const int token = ctid;
                    const bool ok = seen(it, ctx_hi, pos0 + token);
                    const float* kp = reinterpret_cast<const float*>(raw_k + (token / BS) * Smem::RSTRIDE + BS * kD);
                    const float ksf = __half2float(f2h(kp[token % BS]));
                    __half zh, zm, zl;
                    split3(ok ? -(ksf * kp[BS + token % BS]) : 0.f, zh, zm, zl);
                    const __half zero = __ushort_as_half(0);
                    *reinterpret_cast<uint4*>(sm.kx[st] + plain16(token, 0)) = make_uint4(h2_bits(zh, zm), h2_bits(zl, zh), h2_bits(zm, zero), 0u);
                    *reinterpret_cast<uint4*>(sm.kx[st] + plain16(token, 1)) = make_uint4(0u, 0u, 0u, 0u);
                }
                tc05::fence_proxy_async_smem();
                warp_arrive(&sm.k_full[st]);
                if (cwarp == 0) PA_TRACE(2, 2, t);

                if (use > 0 && !wait_warp(&sm.v_free[st], (use - 1) & 1, 2)) goto done;
                if (cwarp == 0) PA_TRACE(2, 3, t);
                // this warp's table of (scale, -1024 * scale) for the tile's token pairs
                __syncwarp();
                float vs0 = 0.f, vs1 = 0.f;
                {
                    const int t0k = 2 * lane, t1k = 2 * lane + 1;
                    if (seen(it, ctx_hi, pos0 + t0k)) vs0 = *reinterpret_cast<const float*>(raw_v + (t0k / BS) * Smem::RSTRIDE + BS * kD + 4 * (t0k % BS));
                    if (seen(it, ctx_hi, pos0 + t1k)) vs1 = *reinterpret_cast<const float*>(raw_v + (t1k / BS) * Smem::RSTRIDE + BS * kD + 4 * (t1k % BS));
                }
                const uint32_t s2 = pack_h2(vs0, vs1);
                sm.v_tab[cwarp][lane] = make_uint2(s2, hmul2_bits(s2, 0xE400E400u));
                const bool big = __any_sync(0xffffffffu, !(fabsf(vs0) < 32.f) || !(fabsf(vs1) < 32.f));
                __syncwarp();
                // V'^T = byte * f16(v scale): unit = 16 tokens of one dim
                const int tg = ctid & 3;
                uint2 tab[8];
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const uint4 t4 = *reinterpret_cast<const uint4*>(&sm.v_tab[cwarp][8 * tg + k]);
                    tab[k] = make_uint2(t4.x, t4.y);
                    tab[k + 1] = make_uint2(t4.z, t4.w);
                }
                constexpr int UPR = BS / 16;   // 16-token units per record
#pragma unroll
                for (int i = 0; i < kD / 32; ++i) {
                    const int d = (ctid >> 2) + 32 * i;
                    uint4 lo4, hi4;
                    bytes16_to_h(*reinterpret_cast<const uint4*>(raw_v + (tg / UPR) * Smem::RSTRIDE + d * BS + 16 * (tg % UPR)), lo4, hi4);
                    uint32_t w[8] = {lo4.x, lo4.y, lo4.z, lo4.w, hi4.x, hi4.y, hi4.z, hi4.w};
                    if (!big) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = hfma2_bits(w[k], tab[k].x, tab[k].y);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = hmul2_bits(hadd2_bits(w[k], 0xE400E400u), tab[k].x);
                    }
                    *reinterpret_cast<uint4*>(sm.vt[st] + sw128(d, 2 * tg)) = make_uint4(w[0], w[1], w[2], w[3]);
                    *reinterpret_cast<uint4*>(sm.vt[st] + sw128(d, 2 * tg + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
                }
                if (ctid < kKv) {
                    const int token = ctid;
                    const bool ok = seen(it, ctx_hi, pos0 + token);
                    const float* vp = reinterpret_cast<const float*>(raw_v + (token / BS) * Smem::RSTRIDE + BS * kD);
                    const float vsf = __half2float(f2h(vp[token % BS]));
                    __half zh, zm, zl;
                    split3(ok ? vsf * vp[BS + token % BS] : 0.f, zh, zm, zl);
                    const uint32_t off = (token & 7) * 2;
                    uint8_t* vt = sm.vt[st];
                    *reinterpret_cast<__half*>(vt + sw128(kD + 0, token >> 3) + off) = zh;
                    *reinterpret_cast<__half*>(vt + sw128(kD + 1, token >> 3) + off) = zm;
                    *reinterpret_cast<__half*>(vt + sw128(kD + 2, token >> 3) + off) = zl;
                    *reinterpret_cast<__half*>(vt + sw128(kD + 3, token >> 3) + off) = __ushort_as_half(ok ? (unsigned short)0x3C00u : (unsigned short)0u);
                }
                tc05::fence_proxy_async_smem();
                warp_arrive(&sm.v_full[st]);
                warp_arrive(&sm.raw_free[st]);
                if (cwarp == 0) PA_TRACE(2, 4, t);
            }
        }
        } else {
            if constexpr (MK) {
            // ---- 16-bit caches, masked: the loader's tensor copies bring the tiles; of those that no row sees as a whole, these warps clear the value rows
            // that no row sees (0 times what is not a number is none), of blocks that were not brought too.  (Their keys' logits are not looked at.)
            (void)cwarp;
            constexpr int CH = kD / 8, TP = kConvWarps * 32 / CH, NU = kKv / TP;   // chunks of a row, tokens per pass, passes
            const int ch = ctid % CH, trow = ctid / CH;
            uint32_t t = 0;   // tiles so far
            for (uint32_t ik = 0;; ++ik) {
                It it;
                const int item = fetch_item(ik, it);
                if (item == -2) goto done;
                if (item < 0) break;
                const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
                for (int j = 0; j < it.ntiles; ++j, ++t) {
                    const int pos0 = tile_pos(it, j), st = t % NST;
                    if (!wait_warp(&sm.v_land[st], (t / NST) & 1, 2)) goto done;   // (of every tile: a phase that is not waited for is mistaken for the one two on)
                    if (whole_tile(it, ctx_hi, pos0)) continue;
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const int token = trow + TP * u;
                        if (!seen(it, ctx_hi, pos0 + token))
                            *reinterpret_cast<uint4*>(sm.vt[st] + (uint32_t)(ch >> 3) * (kKv * 128) + sw128(token, ch & 7)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    tc05::fence_proxy_async_smem();
                    warp_arrive(&sm.v_full[st]);
                }
            }
            } else {
            // ---- f16 cache: token rows -> operand tiles with cp.async; thread = 16-byte chunk `ch` of the rows trow + TP u.
            // The copies of tile t are in flight while tile t - 1 is handed over: K_t is issued, then K_(t-1) is
            // awaited, fenced for the tensor core's proxy and published, then the same for V.
            (void)cwarp;
            constexpr int CH = kD / 8, TP = kConvWarps * 32 / CH, NU = kKv / TP;   // chunks of a row, tokens per pass, passes
            const int ch = ctid % CH, trow = ctid / CH;
            const uint32_t dst0 = (uint32_t)(ch >> 3) * (kKv * 128);
            uint32_t t = 0;
            bool bad_index = false;
            for (uint32_t ik = 0;; ++ik) {
                It it;
                const int item = fetch_item(ik, it);
                if (item == -2) goto done;
                if (item < 0) break;
                const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
                const uint8_t* kc = (const uint8_t*)a.key_cache + (long long)it.hk * a.g.head_bytes + 16 * ch;
                const uint8_t* vc = (const uint8_t*)a.value_cache + (long long)it.hk * a.g.head_bytes + 16 * ch;
                for (int j = 0; j < it.ntiles; ++j, ++t) {
                    const int st = t % NST, stp = (t + NST - 1) % NST;
                    const uint32_t use = t / NST;
                    const int pos0 = tile_pos(it, j);
                    long long off[NU];   // byte offset of this thread's chunk of token trow + TP u; -1: beyond the context
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const int token = trow + TP * u;
                        off[u] = -1;
                        if (seen(it, ctx_hi, pos0 + token)) {
                            int blk = it.table[pos0 / BS + token / BS];
                            if (blk < 0 || blk >= a.num_blocks) { blk = 0; bad_index = true; }
                            off[u] = (long long)blk * a.g.block_bytes + (long long)(token % BS) * (kD * 2);
                        }
                    }
                    if (use > 0 && !wait_warp(&sm.k_free[st], (use - 1) & 1, 1)) goto done;
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const bool ok = off[u] >= 0;
                        cp_async16_zfill(sm.k[st] + dst0 + sw128(trow + TP * u, ch & 7), kc + (ok ? off[u] : 0), ok ? 16u : 0u);
                    }
                    cp_async_commit();
                    if (t > 0) {
                        cp_async_wait<2>();   // pending at most V_(t-1), K_t
                        tc05::fence_proxy_async_smem();
                        warp_arrive(&sm.k_full[stp]);
                    }
                    if (use > 0 && !wait_warp(&sm.v_free[st], (use - 1) & 1, 2)) goto done;
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const bool ok = off[u] >= 0;
                        cp_async16_zfill(sm.vt[st] + dst0 + sw128(trow + TP * u, ch & 7), vc + (ok ? off[u] : 0), ok ? 16u : 0u);
                    }
                    cp_async_commit();
                    if (t > 0) {
                        cp_async_wait<2>();   // pending at most K_t, V_t
                        tc05::fence_proxy_async_smem();
                        warp_arrive(&sm.v_full[stp]);
                    }
                }
            }
            if (t > 0) {
                cp_async_wait<1>();
                tc05::fence_proxy_async_smem();
                warp_arrive(&sm.k_full[(t - 1) % NST]);
                cp_async_wait<0>();
                tc05::fence_proxy_async_smem();
                warp_arrive(&sm.v_full[(t - 1) % NST]);
            }
            if (__any_sync(0xffffffffu, bad_index) && lane == 0) atomicOr(a.status, PA_DEV_BAD_BLOCK_INDEX);
            }
        }
    } else if (warp == kWarpMma || (TwoMma && warp == kWarpMma2)) {
        // ======================= mma issue ================================================================
        // u8 cache: one warp serves both halves in turn, S of tile j + 1 of a half behind P of its tile j.  16-bit caches: one warp
        // per half, so that neither half's waits hold up the other's instructions, and S of tile j + 1 is issued as soon as
        // the softmax warps hold S of tile j in registers; nine ragged bf16 prompts 214 -> 202 us.  Over the u8 cache that was
        // slower (716 -> 765 us on 16 x 512; two warps with the later S 771): both halves then wait for the converter's
        // tile together and their exponentials, which took turns on the special function unit, meet there.
        // The whole warp runs the loop (uniform control flow keeps the descriptors in uniform registers);
        // one elected lane issues the tensor-core instructions.
        {
            constexpr uint32_t idesc_s = tc05::instr_desc_f16(kRows, kKv, kFmt, 0, 0);   // A and B K-major
            constexpr uint32_t idesc_o = U8 ? tc05::instr_desc_f16(kRows, kNo, 0, 0, 0) : tc05::instr_desc_f16(kRows, kD, kFmt, 0, 1);   // f16 / bf16 cache: V' MN-major
            constexpr uint32_t idesc_l = tc05::instr_desc_f16(kRows, kDx, 0, 0, 0);   // f16 cache: P . ones
            // operand descriptors are built once; a step along K or to another buffer only moves the
            // start-address field (bits [0,14) of the low word, in 16-byte units, no carry out of it)
            const uint64_t dq = tc05::smem_desc_sw128(smem_u32(sm.q[0]), 1024), dk = tc05::smem_desc_sw128(smem_u32(sm.k[0]), 1024);
            // MN-major V' of the f16 cache: 8-token groups 1024 bytes apart, the two 64-dim atoms kKv * 128 bytes apart
            const uint64_t dv = U8 ? tc05::smem_desc_sw128(smem_u32(sm.vt[0]), 1024) : tc05::smem_desc_sw128(smem_u32(sm.vt[0]), 1024, kKv * 128);
            uint64_t dqx = 0, dkx = 0, dones = 0;
            uint32_t qx_step = 0, kx_step = 0;
            if constexpr (U8) {
                dqx = tc05::smem_desc_plain(smem_u32(sm.qx[0]), 128, 256);
                dkx = tc05::smem_desc_plain(smem_u32(sm.kx[0]), 128, 256);
                qx_step = sizeof(sm.qx[0]) >> 4;
                kx_step = sizeof(sm.kx[0]) >> 4;
            } else if constexpr (!BF) {
                dones = tc05::smem_desc_plain(smem_u32(sm.ones), 128, 256);
            }
            constexpr uint32_t q_step = sizeof(sm.q[0]) >> 4, k_step = sizeof(sm.k[0]) >> 4, v_step = sizeof(sm.vt[0]) >> 4;
            auto issue_s = [&](int X, int st) {
                const uint64_t da0 = dq + X * q_step, db0 = dk + st * k_step;
                const uint32_t d = tmem + kKv * X;
                if (tc05::elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kD / 16; ++kk) {
                    const uint32_t a_off = ((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4, b_off = ((kk >> 2) * (kKv * 128) + (kk & 3) * 32) >> 4;
                    if (kk == 0) tc05::mma_ss<0>(d, da0 + a_off, db0 + b_off, idesc_s);
                    else tc05::mma_ss<1>(d, da0 + a_off, db0 + b_off, idesc_s);
                }
                if constexpr (U8) tc05::mma_ss<1>(d, dqx + X * qx_step, dkx + st * kx_step, idesc_s);
                tc05::commit(&sm.s_full[X]);
                }
                __syncwarp();
            };
            auto issue_pv = [&](int X, int st, bool acc) {
                const uint32_t pa = tmem + kTmemP + kPCols * X;   // 16 tokens of P = 8 columns
                const uint64_t db0 = dv + st * v_step;
                const uint32_t d = tmem + 2 * kKv + kNo * X;
                if (tc05::elect_one()) {
                if constexpr (U8) {
                    if (acc) tc05::mma_ts<1>(d, pa, db0, idesc_o);
                    else tc05::mma_ts<0>(d, pa, db0, idesc_o);
#pragma unroll
                    for (int kk = 1; kk < kKv / 16; ++kk) tc05::mma_ts<1>(d, pa + 8 * kk, db0 + 2 * kk, idesc_o);
                } else if constexpr (BF) {
                    // high pieces of P, then the low pieces against the same value rows
                    if (acc) tc05::mma_ts<1>(d, pa, db0, idesc_o);
                    else tc05::mma_ts<0>(d, pa, db0, idesc_o);
#pragma unroll
                    for (int kk = 1; kk < kKv / 16; ++kk) tc05::mma_ts<1>(d, pa + 8 * kk, db0 + 128 * kk, idesc_o);
#pragma unroll
                    for (int kk = 0; kk < kKv / 16; ++kk) tc05::mma_ts<1>(d, pa + kKv / 2 + 8 * kk, db0 + 128 * kk, idesc_o);
                } else {
                    // 16 tokens further along K = 16 rows of 128 bytes; the denominators go to the 16 columns after O
                    if (acc) { tc05::mma_ts<1>(d, pa, db0, idesc_o); tc05::mma_ts<1>(d + kD, pa, dones, idesc_l); }
                    else { tc05::mma_ts<0>(d, pa, db0, idesc_o); tc05::mma_ts<0>(d + kD, pa, dones, idesc_l); }
#pragma unroll
                    for (int kk = 1; kk < kKv / 16; ++kk) {
                        tc05::mma_ts<1>(d, pa + 8 * kk, db0 + 128 * kk, idesc_o);
                        tc05::mma_ts<1>(d + kD, pa + 8 * kk, dones, idesc_l);
                    }
                }
                tc05::commit(&sm.o_done[X]);
                }
                __syncwarp();
            };
            uint32_t t = 0;   // tiles so far, over all items
            if constexpr (!TwoMma) {
                uint32_t n[2] = {0, 0}, iq[2] = {0, 0};
                for (uint32_t ik = 0;; ++ik) {
                    It it;
                    const int item = fetch_item(ik, it);
                    if (item == -2) goto done;
                    if (item < 0) break;
                    // first S of the item.  The S region of a half is free: its softmax published the last P of
                    // the previous item (waited below) after reading that tile's S.
                    if (!wait_warp(&sm.k_full[t % NST], (t / NST) & 1, 1)) goto done;
#pragma unroll
                    for (int X = 0; X < 2; ++X)
                        if (it.nt[X] > 0) {
                            if (!wait_warp(&sm.q_full[X], iq[X] & 1, 0)) goto done;
                            ++iq[X];
                            tc05::fence_after_thread_sync();
                            issue_s(X, t % NST);
                        }
                    if (tc05::elect_one()) tc05::commit(&sm.k_free[t % NST]);
                    for (int j = 0; j < it.ntiles; ++j, ++t) {
                        const int st = t % NST, st1 = (t + 1) % NST;
                        const bool more = j + 1 < it.ntiles;
                        PA_TRACE(3, 0, t);
                        // The converter finishes V' of tile j before K' of tile j + 1, so the latter's barrier
                        // covers both; only the item's last tile waits for its V' directly.
                        if (more) {
                            if (!wait_warp(&sm.k_full[st1], ((t + 1) / NST) & 1, 1)) goto done;
                        } else {
                            if (!wait_warp(&sm.v_full[st], (t / NST) & 1, 3)) goto done;
                        }
                        PA_TRACE(3, 3, t);
#pragma unroll
                        for (int X = 0; X < 2; ++X)
                            if (j < it.nt[X]) {
                                // P of tile j is in TMEM, so S of tile j has been read: both MMAs may go
                                if (!wait_warp(&sm.p_full[X], (n[X] + j) & 1, 4)) goto done;
                                PA_TRACE(3, 4 + 2 * X, t);
                                tc05::fence_after_thread_sync();
                                // the next logits first: the half's softmax warps wait for them, nobody waits for this P.V yet
                                if (j + 1 < it.nt[X]) issue_s(X, st1);
                                issue_pv(X, st, j > 0);
                                PA_TRACE(3, 5 + 2 * X, t);
                            }
                        if (tc05::elect_one()) {
                            if (more) tc05::commit(&sm.k_free[st1]);
                            tc05::commit(&sm.v_free[st]);
                        }
                    }
                    n[0] += it.nt[0];
                    n[1] += it.nt[1];
                }
            } else {
                const int X = warp == kWarpMma ? 0 : 1;
                uint32_t n = 0, iq = 0;   // tiles and items of this half
                [[maybe_unused]] uint32_t cleared = 0;   // masked, 16-bit caches: bit s, the phase of v_full[s]
                for (uint32_t ik = 0;; ++ik) {
                    It it;
                    const int item = fetch_item(ik, it);
                    if (item == -2) goto done;
                    if (item < 0) break;
                    const int nt = it.nt[X];
                    [[maybe_unused]] const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
                    // first S of the item.  The S region is free: the half's softmax staged these rows after it had read the last S.
                    if (nt > 0) {
                        if (!wait_warp(&sm.q_full[X], iq & 1, 0)) goto done;
                        ++iq;
                    }
                    // tiles of this half, and a tile's number among them; S runs ahead by one of the half's tiles
                    auto uses = [&](int j) -> bool {
                        if constexpr (MK) return it.uses(X, j);
                        else return j < nt;
                    };
                    auto own = [&](int j) -> int {
                        if constexpr (MK) return it.own(j);
                        else return j;
                    };
                    int ahead = 1;
                    if constexpr (MK) ahead = it.dup ? 2 : 1;
                    for (int j = -ahead; j < it.ntiles; ++j) {
                        if (j >= 0) PA_TRACE(3 + 2 * X, 0, t + j);
                        if (j + ahead < it.ntiles) {
                            const int js = j + ahead, st1 = (t + js) % NST;
                            if (!wait_warp(&sm.k_full[st1], ((t + js) / NST) & 1, 1)) goto done;
                            if (uses(js)) {
                                if (own(js) > 0 && !wait_warp(&sm.s_read[X], (n + own(js) - 1) & 1, 2)) goto done;
                                tc05::fence_after_thread_sync();
                                issue_s(X, st1);
                                if (tc05::elect_one()) tc05::commit(&sm.k_free[st1]);
                                __syncwarp();
                                if (j >= 0) PA_TRACE(3 + 2 * X, 1, t + j);
                            } else {
                                warp_arrive(&sm.k_free[st1]);   // this half has no use for the tile
                            }
                        }
                        if (j >= 0) {
                            const int st = (t + j) % NST;
                            if constexpr (!U8 && MK) {
                                if (whole_tile(it, ctx_hi, tile_pos(it, j))) {
                                    if (!wait_warp(&sm.v_land[st], ((t + j) / NST) & 1, 3)) goto done;
                                } else {
                                    if (!wait_warp(&sm.v_full[st], (cleared >> st) & 1u, 3)) goto done;
                                    cleared ^= 1u << st;
                                }
                            } else {
                                if (!wait_warp(&sm.v_full[st], ((t + j) / NST) & 1, 3)) goto done;
                            }
                            PA_TRACE(3 + 2 * X, 3, t + j);
                            if (uses(j)) {
                                if (!wait_warp(&sm.p_full[X], (n + own(j)) & 1, 4)) goto done;
                                PA_TRACE(3 + 2 * X, 4, t + j);
                                tc05::fence_after_thread_sync();
                                issue_pv(X, st, own(j) > 0);
                                if (tc05::elect_one()) tc05::commit(&sm.v_free[st]);
                                __syncwarp();
                                PA_TRACE(3 + 2 * X, 5, t + j);
                            } else {
                                warp_arrive(&sm.v_free[st]);
                            }
                        }
                    }
                    t += it.ntiles;
                    n += nt;
                }
            }
            // every commit has landed before the CTA's shared memory is given up
            if (t > 0) wait_warp(&sm.v_free[(t - 1) % NST], ((t - 1) / NST) & 1, 0);
        }
    } else if (warp == kWarpLoad) {
        // ======================= loader: TMA-engine copies of the tiles' records =========================
        if (lane == 0) {
            uint32_t t = 0;
            bool bad_index = false;
            std::conditional_t<MK, MaskWalk, int> walk = make_walk<MK>(a);
            for (uint32_t ik = 0;; ++ik) {
                const int slot = ik & (kItemSlots - 1);
                if (ik >= kItemSlots && !wait(&sm.item_free[slot], ((ik / kItemSlots) - 1) & 1, 1)) goto done;
                if constexpr (!U8 && !MK) {
                    // Nothing throttles this loader (it copies no tiles), and an item drawn early is an item another CTA cannot
                    // take: the next one is drawn when every role has started the previous one, which is still several tiles
                    // before the copy warps need it.
                    if (ik >= 1 && !wait(&sm.item_free[(ik - 1) & (kItemSlots - 1)], ((ik - 1) / kItemSlots) & 1, 1)) goto done;
                }
                int item;
                It it{};
                if constexpr (MK) {
                    item = walk.next(a, G, it) ? 0 : -1;
                } else {
                    item = atomicAdd(&a.plan->next_pitem, 1);
                    if (item >= total_items) item = -1;
                    if (item >= 0) it = locate_item(a, item, G, Hkv);
                }
                if (item >= 0) sm.item_desc[slot] = it;
                sm.item_ring[slot] = item;
                mbar_arrive(&sm.item_full[slot]);
                if (item < 0) break;
                const int ctx_hi = max(it.ctx_hi[0], it.ctx_hi[1]);
                // block ids of an item's j-th tile, -1: no row sees any of the block
                [[maybe_unused]] auto look_up = [&](int j, int (&blocks)[Smem::NREC]) {
                    const int pos0 = tile_pos(it, j);
#pragma unroll
                    for (int r = 0; r < Smem::NREC; ++r) {
                        const int bi = pos0 / BS + r;
                        bool any = bi * BS < ctx_hi;
                        if constexpr (MK) any = any && (bi * BS < a.m.sinks || (bi + 1) * BS > it.lo);
                        blocks[r] = any ? it.table[bi] : -1;
                        if (any && (blocks[r] < 0 || blocks[r] >= a.num_blocks)) { blocks[r] = 0; bad_index = true; }
                    }
                };
                if constexpr (!U8 && MK) {
                    // tensor copies straight into the swizzled operand tiles; all stages under way
                    int next[Smem::NREC];
                    look_up(0, next);
                    for (int j = 0; j < it.ntiles; ++j, ++t) {
                        const int st = t % NST;
                        const uint32_t use = t / NST;
                        int blocks[Smem::NREC];
                        uint32_t bytes = 0;
#pragma unroll
                        for (int r = 0; r < Smem::NREC; ++r) {
                            blocks[r] = next[r];
                            bytes += blocks[r] >= 0 ? BS * kD * 2 : 0;
                        }
                        if (j + 1 < it.ntiles) look_up(j + 1, next);
                        auto bring = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar) {
                            mbar_expect_tx(bar, bytes);
#pragma unroll
                            for (int r = 0; r < Smem::NREC; ++r)
                                if (blocks[r] >= 0) {
#pragma unroll
                                    for (int c = 0; c < kD / 64; ++c) tma_3d(dst + c * (kKv * 128) + r * (BS * 128), map, 64 * c, 0, blocks[r] * Hkv + it.hk, bar);
                                }
                        };
                        if (use > 0 && !wait(&sm.k_free[st], (use - 1) & 1, 0)) goto done;
                        bring(sm.k[st], &a.m.map_k, &sm.k_full[st]);
                        begun = t + 1;
                        if (use > 0 && !wait(&sm.v_free[st], (use - 1) & 1, 0)) goto done;
                        bring(sm.vt[st], &a.m.map_v, &sm.v_land[st]);
                        begun_v = t + 1;
                    }
                }
                if constexpr (U8) {
                const uint8_t* kc = (const uint8_t*)a.key_cache + (long long)it.hk * a.g.head_bytes;
                const uint8_t* vc = (const uint8_t*)a.value_cache + (long long)it.hk * a.g.head_bytes;
                [[maybe_unused]] int next[Smem::NREC];   // masked: the next tile's, looked up before the wait for its stage
                if constexpr (MK) look_up(0, next);
                for (int j = 0; j < it.ntiles; ++j, ++t) {
                    const int st = t & 1;
                    const uint32_t use = t >> 1;
                    int blocks[Smem::NREC];
                    if constexpr (MK) {
#pragma unroll
                        for (int r = 0; r < Smem::NREC; ++r) blocks[r] = next[r];
                        if (j + 1 < it.ntiles) look_up(j + 1, next);
                    }
                    if (use > 0 && !wait(&sm.raw_free[st], (use - 1) & 1, 0)) goto done;
                    PA_TRACE(4, 0, t);
                    if constexpr (!MK) look_up(j, blocks);
                    uint32_t bytes = 0;
#pragma unroll
                    for (int r = 0; r < Smem::NREC; ++r) bytes += blocks[r] >= 0 ? 2 * Smem::REC : 0;
                    mbar_expect_tx(&sm.raw_full[st], bytes);
                    if constexpr (MK) begun = t + 1;
#pragma unroll
                    for (int r = 0; r < Smem::NREC; ++r)
                        if (blocks[r] >= 0) {
                            bulk_g2s(sm.raw_k[st] + r * Smem::RSTRIDE, kc + (long long)blocks[r] * a.g.block_bytes, Smem::REC, &sm.raw_full[st]);
                            bulk_g2s(sm.raw_v[st] + r * Smem::RSTRIDE, vc + (long long)blocks[r] * a.g.block_bytes, Smem::REC, &sm.raw_full[st]);
                        }
                }
                }
            }
            if (bad_index) atomicOr(a.status, PA_DEV_BAD_BLOCK_INDEX);
        }
    }
done:
#ifdef PA_PREFILL_PROF
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        const long long base = trace[3][0][0];   // the first mma warp takes up tile 64
        auto at = [&](int role, int ev, int tl) { return trace[role][ev][tl] ? trace[role][ev][tl] - base : 0; };
        for (int role = 0; role < kTraceRoles && base; ++role)
            for (int tl = 0; tl < 4; ++tl)
                printf("trace role %d tile %d: %lld %lld %lld %lld %lld %lld %lld %lld\n", role, 64 + tl, at(role, 0, tl), at(role, 1, tl), at(role, 2, tl),
                       at(role, 3, tl), at(role, 4, tl), at(role, 5, tl), at(role, 6, tl), at(role, 7, tl));
    }
    if (blockIdx.x == 0 && lane == 0 && (warp == 0 || warp == 4 || warp == kSoftmaxWarps || warp >= kWarpMma))
        printf("prefill prof warp %d total %lld waits %lld %lld %lld %lld %lld\n", warp, clock64() - prof_begin, prof[0], prof[1], prof[2], prof[3], prof[4]);
#endif
    if constexpr (!U8) cp_async_wait<0>();   // an aborted copy warp leaves no copy in flight
    if constexpr (MK) {
        cp_async_wait<0>();
        // nor does the loader
        if (warp == kWarpLoad && lane == 0 && sm.abort) {
            for (uint32_t i = begun > NST ? begun - NST : 0; i < begun; ++i) {
                if constexpr (U8) {
                    mbar_wait_bounded(&sm.raw_full[i % NST], (i / NST) & 1);
                } else {
                    mbar_wait_bounded(&sm.k_full[i % NST], (i / NST) & 1);
                    if (i < begun_v) mbar_wait_bounded(&sm.v_land[i % NST], (i / NST) & 1);
                }
            }
        }
    }
    tc05::fence_before_thread_sync();
    __syncthreads();
    if (warp == 0) tc05::tmem_dealloc(tmem, kTmemCols);
}

}  // namespace

bool prefill_tc_supported(const CacheGeom& g) {
    // the bf16 cache with bf16 activations only: other queries would need a second, low piece of every row
    const bool cache_ok = g.cache == PA_DTYPE_U8 || g.cache == PA_DTYPE_F16 || (g.cache == PA_DTYPE_BF16 && g.act == PA_DTYPE_BF16);
    return cache_ok && (g.D == 128 || g.D == 64) && (g.bs == 32 || g.bs == 16) && g.Hq % g.Hkv == 0;
}

namespace {
template <int BS, int CT, int D, bool MK>
cudaError_t launch_tc_t(const KernelArgs& a, cudaStream_t stream, int grid) {
    const int bytes = (int)sizeof(PrefillSmem<BS, CT, D, MK>) + 1024;
    static_assert(sizeof(PrefillSmem<BS, CT, D, MK>) + 1024 <= 232448, "227 KB a block");
    cudaError_t e = cudaFuncSetAttribute(prefill_tc_kernel<BS, CT, D, MK>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    return launch_dependent(prefill_tc_kernel<BS, CT, D, MK>, dim3(grid), dim3(kThreads), bytes, stream, a);
}
template <int CT, int D, bool MK>
cudaError_t launch_tc_bs(const KernelArgs& a, cudaStream_t stream, int grid) {
    return a.g.bs == 32 ? launch_tc_t<32, CT, D, MK>(a, stream, grid) : launch_tc_t<16, CT, D, MK>(a, stream, grid);
}
template <int CT, int D>
cudaError_t launch_tc_mk(const KernelArgs& a, cudaStream_t stream, int grid) {
    return a.m.on ? launch_tc_bs<CT, D, true>(a, stream, grid) : launch_tc_bs<CT, D, false>(a, stream, grid);
}
}  // namespace

cudaError_t launch_prefill_tc(const KernelArgs& a, cudaStream_t stream, int sm_count, long long max_items, int* launches) {
    if (max_items <= 0) return cudaSuccess;
    const int grid = (int)std::min<long long>(max_items, sm_count);
    cudaError_t e;
    if (a.g.cache == PA_DTYPE_U8) e = a.g.D == 128 ? launch_tc_mk<PA_DTYPE_U8, 128>(a, stream, grid) : launch_tc_mk<PA_DTYPE_U8, 64>(a, stream, grid);
    else if (a.g.cache == PA_DTYPE_F16) e = a.g.D == 128 ? launch_tc_mk<PA_DTYPE_F16, 128>(a, stream, grid) : launch_tc_mk<PA_DTYPE_F16, 64>(a, stream, grid);
    else e = a.g.D == 128 ? launch_tc_mk<PA_DTYPE_BF16, 128>(a, stream, grid) : launch_tc_mk<PA_DTYPE_BF16, 64>(a, stream, grid);
    if (e != cudaSuccess) return e;
    ++*launches;
    return cudaSuccess;
}

}  // namespace pa
