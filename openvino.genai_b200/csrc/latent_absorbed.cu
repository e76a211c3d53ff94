// Latent attention in its absorbed form, on the 5th-generation tensor cores (tcgen05 + TMEM): query rows are moved into the latent space
// (q~ = key_up^T q), attend over the paged latents as they lie in the cache, and the sums of latents go through value_up.
//   project_query   q~ per head, and the plan of the attention (first CTA)
//   attend          split over the context: every CTA an equal slice of all (row tile, context tile) units
//   project_value   joins the partial results of the rows, output per head
#include <algorithm>

#include "latent_tc.cuh"

namespace latent {

namespace {

// ---- the plan --------------------------------------------------------------------------------------------------------
// A run costs about two tiles more than its tiles: its queries come in, nothing overlaps its first S, and its results go out.  They are units of the
// slices like tiles, past the context's end (24 sequences, 96 rows by 16 heads: 50.6 us with none, 48.7 with one, 47.6 with two, 48.4 with three).
constexpr int kRunUnits = 2;
struct SeqPlan {
    int blocks;          // row blocks
    long long tiles;     // units of each: context tiles, then kRunUnits
    int tokens;
};
__device__ __forceinline__ SeqPlan seq_plan(const AbsorbedArgs& a, int s) {
    SeqView v;
    if (!seq_view(a.m, s, v) || v.n == 0 || !takes_absorbed(a.m, v)) return SeqPlan{0, 0, 0};
    const int rows = kTile * a.row_tiles;
    return SeqPlan{(int)(((long long)v.n * a.m.H + rows - 1) / rows), ((long long)v.past + v.n + kTokens - 1) / kTokens + kRunUnits, v.n};
}

// Exclusive prefix sums over the sequences, by one block of 128 threads.
__device__ void build_plan(const AbsorbedArgs& a) {
    __shared__ long long sh_u[4], run_u, sh_t[4], run_t;
    __shared__ int sh_b[4], run_b;
    const Step& m = a.m;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, B = m.num_sequences;
    if (tid == 0) { run_u = run_t = 0; run_b = 0; }
    __syncthreads();
    for (int base = 0; base < B; base += 128) {
        const int s = base + tid;
        const SeqPlan p = s < B ? seq_plan(a, s) : SeqPlan{0, 0, 0};
        long long u = p.blocks * p.tiles, k = p.tokens;
        int b = p.blocks;
        const long long mine_u = u;
        const int mine_b = b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long pu = __shfl_up_sync(0xffffffffu, u, o), pk = __shfl_up_sync(0xffffffffu, k, o);
            const int pb = __shfl_up_sync(0xffffffffu, b, o);
            if (lane >= o) { u += pu; b += pb; k += pk; }
        }
        if (lane == 31) { sh_u[wid] = u; sh_b[wid] = b; sh_t[wid] = k; }
        __syncthreads();
        long long off_u = run_u, off_t = run_t;
        int off_b = run_b;
        for (int w = 0; w < wid; ++w) { off_u += sh_u[w]; off_b += sh_b[w]; off_t += sh_t[w]; }
        if (s < B) { a.unit_prefix[s] = off_u + u - mine_u; a.block_prefix[s] = off_b + b - mine_b; a.token_prefix[s] = (int)(off_t + k - p.tokens); }
        __syncthreads();
        if (tid == 127) { run_u = off_u + u; run_b = off_b + b; run_t = off_t + k; }
        __syncthreads();
    }
    // Prefix sums that fall can give sequences the same tokens, more in all than the workspace has rows for: such a step gets no plan.
    if (tid == 0 && run_t > m.num_tokens) {
        atomicOr(m.status, PA_DEV_BAD_BEGINS);
        run_u = run_t = 0;
    }
    if (tid == 0) { a.unit_prefix[B] = run_u; a.block_prefix[B] = run_b; a.token_prefix[B] = (int)run_t; }
    __syncthreads();
    // where every slice begins, so that a CTA of the attention has one record to read instead of a search
    const long long total = run_u, per = total > 0 ? (total + a.groups - 1) / a.groups : 1;
    for (int w = tid; w < a.groups; w += 128) {
        const long long u = w * per;
        SliceStart st{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        if (u < total) {
            int lo = 0, hi = B;              // unit_prefix[lo] <= u < unit_prefix[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.unit_prefix[mid] <= u) lo = mid; else hi = mid;
            }
            SeqView v;
            seq_view(a.m, lo, v);
            const SeqPlan p = seq_plan(a, lo);
            const long long rel = u - a.unit_prefix[lo];
            st = SliceStart{lo, (int)(rel / p.tiles), (int)(rel % p.tiles), (int)min(per, total - u), v.t0, v.n, v.past, v.tb, p.blocks, (int)p.tiles, a.block_prefix[lo],
                            (int)per};
        }
        a.starts[w] = st;
    }
}

// Which of the tile's tokens belong to sequences of this form; false (for the whole block) if none does.
template <int NT>
__device__ __forceinline__ bool tile_rows(const AbsorbedArgs& a, int t0, bool (&live)[NT]) {
    bool mine = false;
    if (threadIdx.x < NT) {
        SeqView v;
        mine = t0 + (int)threadIdx.x < a.m.num_tokens && token_view(a.m, t0 + threadIdx.x, v) && takes_absorbed(a.m, v);
        live[threadIdx.x] = mine;
    }
    return __syncthreads_or(mine) != 0;
}

// ---- q~ = key_up^T q ----------------------------------------------------------------------------------------------------
// A CTA computes 128 latent elements of 64 tokens of one head: D[latent][token] with the weight's rows (d, latent contiguous) as an
// MN-major operand, one tile of each operand, so the CTAs of an SM overlap one another's loads, products and stores.  q~ is rounded to 16 bits: it is
// an operand of the attention's products.  9 us for one row by 128 heads (34 MB of weights), 6 of them the chain plan -> loads -> product -> stores.
template <bool BF>
__global__ void __launch_bounds__(128) project_query_kernel(const __grid_constant__ AbsorbedArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t full, done, idle;
    __shared__ bool live[kTile];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    const Step& m = a.m;
    if (blockIdx.x == 0) {
        pa::grid_wait();
        pa::grid_release();
        build_plan(a);
        return;
    }
    const int parts = m.R / 128, tid = threadIdx.x, warp = warp_id(), lane = tid & 31;
    const int i = blockIdx.x - 1, part = i % parts, h = i / parts % m.H, t0 = i / parts / m.H * kTile;
    uint8_t* const sw = smem;                        // two atoms of [Dn][64 latent elements]
    uint8_t* const sq = smem + 2 * m.Dn * 128;       // Dn / 64 atoms of [64 tokens][64 elements]
    if (tid == 0) {
        pa::mbar_init(&full, 1);
        pa::mbar_init(&done, 1);
        pa::mbar_init(&idle, 1);
        pa::mbar_fence_init();
        abort_flag = 0;
        for (int c = 0; c < 2; ++c) prefetch_3d(&a.map_key_up, part * 128 + c * 64, 0, h);
    }
    if (warp == 0) tc05::tmem_alloc(&tmem_base, 64);
    pa::grid_wait();
    pa::grid_release();
    if (tid == 0) {
        pa::mbar_expect_tx(&full, 2 * m.Dn * 128 + m.Dn / 64 * 8192);
        for (int c = 0; c < 2; ++c) tma_3d(sw + c * m.Dn * 128, &a.map_key_up, part * 128 + c * 64, 0, h, &full);
        for (int c = 0; c < m.Dn / 64; ++c) tma_3d(sq + c * 8192, &a.map_qn, c * 64, h, t0, &full);
    }
    tc05::fence_before_thread_sync();
    const bool any = tile_rows(a, t0, live);
    tc05::fence_after_thread_sync();
    const Waiter wt{&abort_flag, m.status, m.wait_polls};
    const uint32_t tmem = tmem_base;
    bool ok = wt.wait(&full, 0);
    if (any && warp == 0 && __all_sync(0xffffffffu, ok)) {
        constexpr uint32_t idesc = tc05::instr_desc_f16(128, kTile, BF ? 1 : 0, 1, 0);
        const uint32_t da = desc_low(sw, m.Dn * 128), db = desc_low(sq);
        if (tc05::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
                const uint32_t pa = da + 128 * kk, pb = db + (kk >> 2) * 512 + (kk & 3) * 2;
                if (kk == 0) mma_ss<0>(tmem, pa, pb, idesc);
                else if (kk < 4 || m.Dn == 128) mma_ss<1>(tmem, pa, pb, idesc);
            }
            tc05::commit(&done);
        }
    }
    if (any && part == 0) {   // the rotated part goes along as it is
        const int pieces = m.P / 8;
        for (int u = tid; u < kTile * pieces; u += 128) {
            const int t = t0 + u / pieces, c = u % pieces;
            if (t < m.num_tokens)
                *reinterpret_cast<uint4*>((uint16_t*)a.q_abs + ((long long)t * m.H + h) * (m.R + m.P) + m.R + 8 * c) =
                    *reinterpret_cast<const uint4*>((const uint16_t*)a.q_rope + t * a.qr_token + h * a.qr_head + 8 * c);
        }
    }
    ok = any && ok && wt.wait(&done, 0);
    tc05::fence_after_thread_sync();
    if (__all_sync(0xffffffffu, ok)) {
        uint16_t* dst = (uint16_t*)a.q_abs + ((long long)t0 * m.H + h) * (m.R + m.P) + part * 128 + tid;
#pragma unroll
        for (int c0 = 0; c0 < kTile; c0 += 32) {
            uint32_t r[32];
            tc05::ld_32x32b_x32(tmem + ((uint32_t)(warp * 32) << 16) + c0, r);
            tc05::wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (live[c0 + c]) dst[(long long)(c0 + c) * m.H * (m.R + m.P)] = pack1<BF>(__uint_as_float(r[c]));
        }
    }
    tc05::fence_before_thread_sync();
    __syncthreads();
    if (warp == 0) {
        if (*(volatile int*)&abort_flag) {
            drain(&full, 0);
            drain_products(&idle);
        }
        tc05::tmem_dealloc(tmem, 64);
    }
    (void)lane;
}

// ---- attention over the latents ------------------------------------------------------------------------------------------
// Roles meet through mbarriers only: a loader warp walks the slice and has the TMA engine bring query rows and 64-token tiles of the cache,
// two warps issue the products, four warps (64 rows, 16 a warp) do the softmax, four more rescale O and write results.
//   S[row][token]     = Q~ K^T          M 64, N 64, K R + P; two buffers, so that S of the next tile is computed beside a softmax
//   O^T[latent][row] += K^T P^T         M 128 (R / 128 times), N 64, K 64: the tile is read MN-major from the same image, and the
//                                       rows (heads) are columns, so few heads leave no tensor-memory lane idle
// A tile lies in shared memory in parts of 128 latent elements, a part in groups of eight tokens, [group][64-element chunk][8 tokens][64]: that is one box of
// a four-dimensional view of the cache.  Two tiles of 512 are all that fits beside the query rows, so the parts come, are multiplied and are freed by
// themselves: one row over 120 k tokens by 128 heads 80.0 us with halves of 32 tokens, 77.5 so.
// S and O are issued by a warp each: one warp for both had to look at two barriers in turn, and a look, with what follows it, is 200 cycles.
// Weights and q~ go in as 16 bits, because both operands of a step have one type; maxima, sums and O are 32 bits, O unscaled until the pieces are joined.
// 64 rows by 128 heads over 259,540 tokens (338 MB): 108 us, tensor pipe 50 % busy, HBM 39 %.  A tile takes 3200 cycles of which the products are 1950; the
// rest is the chain S -> softmax (1150) -> P -> O -> tile free -> load (1500, from the L2 cache) with two tiles in flight.
// Tiles of 32 tokens, four in flight, were no faster: an M 64, N 32 step takes 26 cycles, one of N 64 33.
constexpr int kSlots = 4;               // depth of the queue of runs
constexpr int kThreads = 384;           // warps 0 - 3: softmax, 4: loader, 5: S, 6: O, 8 - 11: rescaling and results (a warp reads the tensor-memory lanes of its number mod 4)
template <int R> constexpr int kAheadOf = R == 512 ? 4 : 6;     // tiles ahead of the loads that are brought into the L2 cache
constexpr float kLazy = 8.f;            // log2 of the growth of a row maximum that rescales O

// A stretch of context tiles of one row tile.
struct Run {
    int rows;            // rows of the tile, 0: no more runs
    int row0;            // its first row among the sequence's (token, head) rows
    long long grow0;     // and among the step's
    int past;
    int first, tiles;    // context tiles
    int end;             // context the tile's last row sees
    int tb;
    int slot;            // of the partial result
    int pieces;          // partial results of the row tile, if this is the first, else 0
};

template <int R>
struct AttendSmem {
    static constexpr int NST = R == 512 ? 2 : 4;    // context tiles in flight
    alignas(1024) uint8_t q[kTile * R * 2];
    alignas(1024) uint8_t q_rope[kTile * 128];
    // A tile is loaded, multiplied and freed in parts of 128 latent elements (64 tokens each), so that the next tile's parts arrive while the
    // others of this one are still being multiplied, and S begins with the first
    static constexpr int NQ = R / 128;
    struct Tile {
        uint8_t c[NQ][kTokens * 256];               // [token / 8][element / 64][token % 8]
        uint8_t rope[kTokens * 128];
    };
    alignas(1024) Tile k[NST];
    alignas(1024) uint8_t p[kTile * 128];           // [row][token]
    float alpha[2][kTile];
    float2 stat[2][kTile];                          // maximum and sum of the rows of a run
    volatile uint32_t grew[2];                      // the last tile (+ 1) in which a row's maximum grew
    volatile int event;                             // what the results warps are asked for: rescale after tile `event` - 1, or results (0)
    uint64_t k_full[NST][NQ], k_free[NST][NQ];      // parts of tiles: loader -> products (bytes), products -> loader
    uint64_t q_full, q_free;
    uint64_t s_full[2], s_free[2];                  // products -> softmax, softmax -> products
    uint64_t p_full, o_done;                        // softmax -> products, products -> softmax and results
    uint64_t asked, answered;                       // products -> results, results -> products
    uint64_t idle[2];                               // after an abort, of the two warps that issue products
    // softmax -> results, runs in turn.  The softmax gets at most a run ahead of the results: a tile's P waits for the products of the tile
    // before, and a run's first products wait for the results of the run before
    uint64_t stat_full[2];
    uint64_t run_full[kSlots], run_free[kSlots];
    Run run[kSlots];
    uint32_t tmem_base;
    int abort_flag;
};

template <int R, bool BF>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const __grid_constant__ AbsorbedArgs a) {
    using Smem = AttendSmem<R>;
    constexpr int NST = Smem::NST, NQ = Smem::NQ, MT = NQ;
    constexpr uint32_t kGroup = 2048;               // bytes from one group of eight tokens of a part to the next
    constexpr uint32_t kPart = kTokens * 256;
    constexpr uint32_t kTmemS = MT * kTile;         // O^T: MT x 64 columns, then S twice
    extern __shared__ __align__(1024) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const Step& m = a.m;
    const int tid = threadIdx.x, warp = warp_id(), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < NQ * NST; ++i) { pa::mbar_init(&sm.k_full[0][i], 1); pa::mbar_init(&sm.k_free[0][i], 1); }
        pa::mbar_init(&sm.q_full, 1);
        pa::mbar_init(&sm.q_free, 1);
        for (int i = 0; i < 2; ++i) { pa::mbar_init(&sm.s_full[i], 1); pa::mbar_init(&sm.s_free[i], 4); pa::mbar_init(&sm.stat_full[i], 4); pa::mbar_init(&sm.idle[i], 1); }
        pa::mbar_init(&sm.p_full, 4);
        pa::mbar_init(&sm.o_done, 1);
        pa::mbar_init(&sm.asked, 1);
        pa::mbar_init(&sm.answered, 4);
        for (int i = 0; i < kSlots; ++i) { pa::mbar_init(&sm.run_full[i], 1); pa::mbar_init(&sm.run_free[i], 10); }
        pa::mbar_fence_init();
        sm.grew[0] = sm.grew[1] = 0;
        sm.abort_flag = 0;
    }
    if (warp == 5) tc05::tmem_alloc(&sm.tmem_base, 512);
    pa::grid_wait();
    pa::grid_release();
    tc05::fence_before_thread_sync();
    __syncthreads();
    tc05::fence_after_thread_sync();
    const uint32_t tmem = sm.tmem_base;
    const Waiter wt{&sm.abort_flag, m.status, m.wait_polls};
    uint32_t queries = 0, parts = 0;      // loader: query tiles and parts of context tiles that it has asked for
    // The next run of the queue; false: a wait ran out.
    auto fetch = [&](uint32_t n, Run& r) -> bool {
        const int slot = n % kSlots;
        if (!wt.wait_warp(&sm.run_full[slot], (n / kSlots) & 1)) return false;
        r = sm.run[slot];
        warp_arrive(&sm.run_free[slot]);
        return true;
    };

    if (warp == 4) {
        // ======================= loader =================================================================
        const int group = blockIdx.x / a.row_tiles, member = blockIdx.x % a.row_tiles;
        const SliceStart start = a.starts[group];
        int s = start.s, block = start.block, first = start.first, left = start.units;     // left: units of the slice
        SeqView v{start.t0, start.n, start.past, start.tb};
        int blocks = start.blocks, tiles = start.tiles, block0 = start.block0;
        uint32_t n = 0, nr = 0;              // tiles, queue entries so far
        const uint64_t policy = evict_first();
        bool ok = true, bad_index = false;
        auto publish = [&](const Run& r) -> bool {
            const int slot = nr % kSlots;
            if (nr >= kSlots && !wt.wait_warp(&sm.run_free[slot], (nr / kSlots - 1) & 1)) return false;
            if (lane == 0) sm.run[slot] = r;
            warp_arrive(&sm.run_full[slot]);
            ++nr;
            return true;
        };
        while (ok && s >= 0 && left > 0) {
            if (block >= blocks) {      // the next sequence with work
                ++s;
                block = first = 0;
                seq_view(m, s, v);
                const SeqPlan plan = seq_plan(a, s);
                blocks = plan.blocks;
                tiles = (int)plan.tiles;
                block0 = a.block_prefix[s];
                continue;
            }
            const int len = min(tiles - first, left);
            Run r;
            r.row0 = (block * a.row_tiles + member) * kTile;
            r.rows = (int)min((long long)kTile, (long long)v.n * m.H - r.row0);
            if (r.rows > 0) {
                r.grow0 = (long long)v.t0 * m.H + r.row0;
                r.past = v.past;
                r.end = v.past + (r.row0 + r.rows - 1) / m.H + 1;
                r.first = first;
                r.tiles = max(0, min(first + len, (r.end + kTokens - 1) / kTokens) - first);
                r.tb = v.tb;
                r.slot = (block0 + block + group) * a.row_tiles + member;
                // the block's units run on through the slices behind this one
                r.pieces = first > 0 ? 0 : 1 + max(0, tiles - left + start.per - 1) / start.per;
                ok = publish(r);
                if (ok && r.tiles > 0) {
                    if (queries > 0) ok = wt.wait_warp(&sm.q_free, (queries - 1) & 1);
                    if (ok && tc05::elect_one()) {
                        pa::mbar_expect_tx(&sm.q_full, kTile * (R * 2 + 128));     // (rows behind the tile's are other rows' or zeros)
                        tma_3d(sm.q, &a.map_q_abs, 0, (int)r.grow0, 0, &sm.q_full);
                        tma_2d(sm.q_rope, &a.map_q_abs_rope, 0, (int)r.grow0, &sm.q_full);
                    }
                    __syncwarp();
                    queries += ok;
                    // pieces of a half tile: 32 tokens of a block, or two blocks of 16 (all powers of two)
                    const int bs_log2 = 31 - __clz(m.bs), piece_log2 = min(bs_log2, 5), piece = 1 << piece_log2, pieces = 32 >> piece_log2;
                    const int sub_log2 = bs_log2 - piece_log2, last_piece = (r.end - 1) >> piece_log2;
                    int page = 0, base = -1;     // this lane's block of the 32 from `base`
                    // group of eight tokens of the cache at which piece `at` of the sequence lies
                    auto group_of = [&](int at) {
                        return (__shfl_sync(0xffffffffu, page, (at >> sub_log2) - base) << (bs_log2 - 3)) + ((at & ((1 << sub_log2) - 1)) << (piece_log2 - 3));
                    };
                    for (int j = 0; ok && j < r.tiles; ++j, ++n) {
                        const int p0 = (r.first + j) * 2 * pieces, b0 = p0 >> sub_log2;
                        if (base < 0 || b0 + (kAheadOf<R> + 1) * 2 * pieces > base + 32) {
                            base = b0;
                            page = 0;
                            if (base + lane <= last_piece >> sub_log2) {
                                page = m.block_indices[r.tb + base + lane];
                                if (page < 0 || page >= m.num_blocks) { page = 0; bad_index = true; }
                            }
                        }
                        const int st = n % NST;
                        int group[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) group[i] = group_of(min(p0 + min(i, 2 * pieces - 1), last_piece));
                        const int count = min(2 * pieces, last_piece - p0 + 1);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            if (n >= NST) ok = ok && wt.wait_warp(&sm.k_free[st][q], (n / NST - 1) & 1);
                            if (!ok) break;
                            if (tc05::elect_one()) {
                                pa::mbar_expect_tx(&sm.k_full[st][q], count * piece * (q + 1 == NQ ? 256 + 128 : 256));
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (i < count) {
                                        tma_4d(sm.k[st].c[q] + i * piece * 256, &a.map_cache_part, 0, 0, 2 * q, group[i], &sm.k_full[st][q], policy);
                                        if (q + 1 == NQ) tma_3d(sm.k[st].rope + i * piece * 128, &a.map_cache_rope, 0, 0, group[i], &sm.k_full[st][q], policy);
                                    }
                            }
                            __syncwarp();
                            ++parts;
                        }
                        // tiles to come go to the L2 cache meanwhile (the CTAs of a group take turns): two tiles in flight do not cover the memory's latency
                        for (int ahead = j == 0 ? NST : kAheadOf<R>; ahead <= kAheadOf<R>; ++ahead)
                            if ((j + ahead) % a.row_tiles == member)
                                for (int i = 0; i < 2 * pieces; ++i) {
                                    const int at = p0 + ahead * 2 * pieces + i, g = group_of(min(at, last_piece));
                                    if (at <= last_piece && tc05::elect_one()) {
                                        prefetch_4d(&a.map_cache, 0, 0, 0, g, policy);
                                        prefetch_3d(&a.map_cache_rope, 0, 0, g, policy);
                                    }
                                    __syncwarp();
                                }
                    }
                }
            }
            left -= len;
            first += len;
            if (first == tiles) { first = 0; ++block; }
        }
        if (ok) {
            Run r{};
            publish(r);
        }
        if (__any_sync(0xffffffffu, bad_index) && lane == 0) atomicOr(m.status, PA_DEV_BAD_BLOCK_INDEX);
    } else if (warp == 5) {
        // ======================= S ========================================================================
        // (the whole warp runs the loop and one elected lane issues: in code that a single lane runs, an instruction took twice as long to issue)
        constexpr uint32_t idesc_s = tc05::instr_desc_f16(kTile, kTokens, BF ? 1 : 0, 0, 0);
        const uint32_t dq = desc_low(sm.q), dqr = desc_low(sm.q_rope), dk = desc_low(sm.k[0].c), dkr = desc_low(sm.k[0].rope);
        constexpr uint32_t kStage = sizeof(typename Smem::Tile) >> 4;
        const bool wide = m.P == 64;
        uint32_t n = 0;
        bool ok = true;
        Run r;
        for (uint32_t nr = 0, nq = 0; ok; ++nr) {
            if (!fetch(nr, r) || r.rows == 0) break;
            if (r.tiles == 0) continue;
            ok = wt.wait_warp(&sm.q_full, nq & 1);
            ++nq;
            for (int j = 0; ok && j < r.tiles; ++j, ++n) {
                const int st = n % NST;
                ok = n < 2 || wt.spin_warp(&sm.s_free[n & 1], ((n >> 1) - 1) & 1);
                const uint32_t db = dk + st * kStage, dbr = dkr + st * kStage, d = tmem + kTmemS + (n & 1) * kTokens;
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    ok = ok && wt.spin_warp(&sm.k_full[st][q], (n / NST) & 1);
                    if (!ok) break;
                    tc05::fence_after_thread_sync();
                    if (tc05::elect_one()) {
#pragma unroll
                        for (int c = 2 * q; c < 2 * q + 2; ++c) {
                            const uint32_t qa = dq + c * (kTile * 128 >> 4), kb = db + q * (kPart >> 4) + (c & 1) * (1024 >> 4);
                            if (c == 0) mma_ss<0, 1024, kGroup>(d, qa, kb, idesc_s);
                            else mma_ss<1, 1024, kGroup>(d, qa, kb, idesc_s);
#pragma unroll
                            for (int kk = 1; kk < 4; ++kk) mma_ss<1, 1024, kGroup>(d, qa + kk * 2, kb + kk * 2, idesc_s);
                        }
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (tc05::elect_one()) {
                    mma_ss<1>(d, dqr, dbr, idesc_s);
                    mma_ss<1>(d, dqr + 2, dbr + 2, idesc_s);
                    if (wide) {
                        mma_ss<1>(d, dqr + 4, dbr + 4, idesc_s);
                        mma_ss<1>(d, dqr + 6, dbr + 6, idesc_s);
                    }
                    tc05::commit(&sm.s_full[n & 1]);
                    if (j + 1 == r.tiles) tc05::commit(&sm.q_free);
                }
                __syncwarp();
            }
        }
    } else if (warp == 6) {
        // ======================= O ========================================================================
        constexpr uint32_t idesc_o = tc05::instr_desc_f16(128, kTile, BF ? 1 : 0, 1, 0);
        const uint32_t dv = desc_low(sm.k[0].c, 1024), dp = desc_low(sm.p);
        constexpr uint32_t kStage = sizeof(typename Smem::Tile) >> 4;
        uint32_t n = 0, asked = 0;
        bool ok = true;
        Run r;
        auto ask = [&](int event) {
            if (lane == 0) sm.event = event;
            warp_arrive(&sm.asked);
            ++asked;
        };
        for (uint32_t nr = 0; ok; ++nr) {
            if (!fetch(nr, r) || r.rows == 0) break;
            if (r.tiles == 0) continue;
            for (int j = 0; ok && j < r.tiles; ++j, ++n) {
                ok = wt.spin_warp(&sm.p_full, n & 1);
                if (ok && j > 0 && sm.grew[n & 1] == n + 1) ask((int)n);
                // (the first product overwrites O: the results of the run before have been read)
                if (ok && asked > 0 && (j == 0 || sm.grew[n & 1] == n + 1)) ok = wt.wait_warp(&sm.answered, (asked - 1) & 1);
                if (!ok) break;
                tc05::fence_after_thread_sync();
                const uint32_t da = dv + n % NST * kStage;
                if (tc05::elect_one()) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const uint32_t d = tmem + mt * kTile;
#pragma unroll
                        for (int kk = 0; kk < kTokens / 16; ++kk) {
                            const uint32_t pa = da + mt * (kPart >> 4) + kk * (2 * kGroup >> 4);
                            if (kk == 0 && j == 0) mma_ss<0, kGroup>(d, pa, dp, idesc_o);
                            else mma_ss<1, kGroup>(d, pa, dp + kk * 2, idesc_o);
                        }
                        tc05::commit(&sm.k_free[n % NST][mt]);
                    }
                    tc05::commit(&sm.o_done);
                }
                __syncwarp();
            }
            if (ok) ask(-1);
        }
    } else if (warp >= 8) {
        // ======================= rescaling and results ====================================================
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int e = 32 * (warp & 3) + lane;           // latent element, of every 128
        uint32_t n = 0, asked = 0;                      // tiles before this run, requests so far
        Run r;
        bool ok = true;
        for (uint32_t nr = 0, ns = 0; ok; ++nr) {
            if (!fetch(nr, r) || r.rows == 0) break;
            for (; r.tiles > 0; ++asked) {
                if (!wt.wait_warp(&sm.asked, asked & 1)) { ok = false; break; }
                const int event = sm.event;
                const uint32_t done = event >= 0 ? (uint32_t)event - 1 : n + r.tiles - 1;    // the products that have to be complete
                if (!wt.wait_warp(&sm.o_done, done & 1)) { ok = false; break; }
                tc05::fence_after_thread_sync();
                if (event < 0) break;
                const float* alpha = sm.alpha[event & 1];
#pragma unroll 1
                for (int q = 0; q < MT * 2; ++q) {
                    uint32_t o[32];
                    tc05::ld_32x32b_x32(tmem + 32 * q + lanes, o);
                    tc05::wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha[(q & 1) * 32 + c]);
                    tc05::st_32x32b_x32(tmem + 32 * q + lanes, o);
                }
                tc05::wait_st();
                tc05::fence_before_thread_sync();
                warp_arrive(&sm.answered);
            }
            if (!ok) break;
            n += r.tiles;
            if (r.pieces > 0 && e < r.rows) a.row_part[r.grow0 + e] = make_int2(r.slot * kTile + e, r.pieces);
            if (r.tiles == 0) {
                if (e < r.rows) a.part_ml[(long long)r.slot * kTile + e] = make_float2(-INFINITY, 0.f);
                continue;
            }
            if (!wt.wait_warp(&sm.stat_full[ns & 1], (ns >> 1) & 1)) break;
            const float2* stat = sm.stat[ns & 1];
            ++ns;
            if (e < r.rows) a.part_ml[(long long)r.slot * kTile + e] = stat[e];
#pragma unroll 1
            for (int q = 0; q < MT * 2; ++q) {
                const int c0 = (q & 1) * 32;
                if (c0 >= r.rows) continue;
                uint32_t o[32];
                tc05::ld_32x32b_x32(tmem + 32 * q + lanes, o);
                tc05::wait_ld();
                float* dst = a.part_o + ((long long)r.slot * kTile + c0) * R + (q >> 1) * 128 + e;
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (c0 + c < r.rows) dst[c * R] = __uint_as_float(o[c]);
            }
            tc05::fence_before_thread_sync();
            warp_arrive(&sm.answered);
            ++asked;
        }
    } else if (warp < 4) {
        // ======================= softmax ==================================================================
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const int rl[2] = {16 * warp + lane / 4, 16 * warp + lane / 4 + 8};     // this thread's rows of S
        const float c2 = a.scale_log2;
        uint32_t n = 0, nst = 0;
        Run r;
        for (uint32_t nr = 0;; ++nr) {
            if (!fetch(nr, r) || r.rows == 0) break;
            int limit[2];          // context each of the thread's two rows sees
            float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 2; ++x) limit[x] = rl[x] < r.rows ? r.past + (r.row0 + rl[x]) / m.H + 1 : 0;
            const int least = __reduce_min_sync(0xffffffffu, min(limit[0], limit[1]));
            bool ok = true;
            for (int j = 0; j < r.tiles; ++j, ++n) {
                if (!wt.wait_warp(&sm.s_full[n & 1], (n >> 1) & 1)) { ok = false; break; }
                tc05::fence_after_thread_sync();
                const bool free_p = n == 0 || mbar_test(&sm.o_done, (n - 1) & 1);      // P of the tile before has been read (looked at early: the answer takes its time)
                uint32_t raw[32];
                ld_16x256b_x8(tmem + kTmemS + (n & 1) * kTokens + lanes, raw);
                tc05::wait_ld();
                tc05::fence_before_thread_sync();
                warp_arrive(&sm.s_free[n & 1]);
                float sv[2][16];
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sv[e >> 1][2 * i + (e & 1)] = __uint_as_float(raw[4 * i + e]);
                const int col0 = (r.first + j) * kTokens;
                if (col0 + kTokens > least) {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (col0 + 8 * (c >> 1) + 2 * (lane & 3) + (c & 1) >= limit[x]) sv[x][c] = -INFINITY;
                }
                bool grew = false;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float t = fmaxf(sv[x][0], sv[x][1]);
#pragma unroll
                    for (int c = 2; c < 16; c += 2) t = max3(t, sv[x][c], sv[x][c + 1]);
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2)) * c2;
                    float alpha = 1.f;
                    // (a row that has seen nothing yet takes its first maximum without a rescale: its O is zero)
                    if (mx[x] == -INFINITY) mx[x] = t;
                    else if (t > mx[x] + kLazy) { alpha = ex2(mx[x] - t); mx[x] = t; grew = true; }
                    if ((lane & 3) == 0) sm.alpha[n & 1][rl[x]] = alpha;
                    l[x] *= alpha;
                    const float ref = mx[x] == -INFINITY ? 0.f : -mx[x];
                    float sum[2] = {0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        sv[x][c] = ex2(fmaf(sv[x][c], c2, ref));
                        sum[c & 1] += sv[x][c];
                    }
                    l[x] += sum[0] + sum[1];
                }
                if (grew) sm.grew[n & 1] = n + 1;
                if (!__all_sync(0xffffffffu, free_p) && !wt.wait_warp(&sm.o_done, (n - 1) & 1)) { ok = false; break; }
                // P: a row's 64 tokens are 128 bytes, 16-byte pieces swizzled by the row
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint32_t*>(sm.p + rl[x] * 128 + ((i ^ (rl[x] & 7)) << 4) + (lane & 3) * 4) = pack2<BF>(sv[x][2 * i], sv[x][2 * i + 1]);
                if (col0 + kTokens > r.end) {
                    // tokens behind the context: whatever lies there (stale bytes, not-a-number) meets probabilities of zero, which does not
                    // make it zero, so the latents are cleared
                    const int st = n % NST, valid = r.end - col0;
                    for (int q = 0; ok && q < NQ; ++q) ok = wt.wait_warp(&sm.k_full[st][q], (n / NST) & 1);
                    if (!ok) break;
                    for (int i = tid; i < (kTokens - valid) * 8; i += 128) {
                        const int row = valid + i / 8;
#pragma unroll
                        for (int c = 0; c < 2 * NQ; ++c)
                            *reinterpret_cast<uint4*>(sm.k[st].c[c >> 1] + (row >> 3) * kGroup + (c & 1) * 1024 + (row & 7) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                tc05::fence_proxy_async_smem();
                tc05::fence_before_thread_sync();
                warp_arrive(&sm.p_full);
            }
            if (!ok) break;
            if (r.tiles == 0) continue;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
                if ((lane & 3) == 0) sm.stat[nst & 1][rl[x]] = make_float2(mx[x], l[x]);
            }
            warp_arrive(&sm.stat_full[nst & 1]);
            ++nst;
        }
    }
    __syncthreads();
    if (*(volatile int*)&sm.abort_flag) {
        if (warp == 4) {
            constexpr uint32_t kParts = NST * NQ;
            if (queries > 0) drain(&sm.q_full, (queries - 1) & 1);
            for (uint32_t i = parts > kParts ? parts - kParts : 0; i < parts; ++i) drain(&sm.k_full[0][0] + i % kParts, (i / kParts) & 1);
        } else if (warp == 5 || warp == 6) drain_products(&sm.idle[warp - 5]);
        __syncthreads();
    }
    if (warp == 5) tc05::tmem_dealloc(tmem, 512);
}

// ---- output = value_up o~ ---------------------------------------------------------------------------------------------------
// A CTA joins the partial results of one head's rows of NT tokens and computes their output: D[value][token], K = R twice, because the joined sums
// go in as two 16-bit pieces (high and low), so that the product does not see another rounding.  Few tokens take tiles of 16, so
// that there are CTAs enough to join their rows.
// Bound by the chain row -> record -> statistics -> partial results -> product -> output, not by the partial results' bytes (22 MB for 96 rows by
// 16 heads of up to 15 pieces, in 7 us).  So a row belongs to a warp from its record to its place in shared memory, with the pieces of the statistics
// dealt over the lanes and the first pieces under way before their weights: the same call took 67.5 us with the pieces of one row after another
// dealt over the block, 50.0 so.  Joining in a kernel of its own took 7 us more than either.
constexpr int kJoinWarps = 16, kJoinThreads = 32 * kJoinWarps;
constexpr int kValueThreads = kJoinThreads + 32;     // warps 0 - 15: joining, then (0 - 3) output; 16: weights and products

template <int R, int NT>
struct ValueSmem {
    static constexpr int NC = R / 64, NW = 4;                    // chunks of 64 latent elements, of which weights are in flight
    alignas(1024) uint8_t o[2][NC][NT * 128];                    // joined rows, high and low pieces
    alignas(1024) uint8_t w[NW][128 * 128];
    uint64_t w_full[NW], w_free[NW], o_full, done, idle;
    int token[NT];
    uint32_t tmem_base;
    int abort_flag;
};

template <int R, int NT, bool BF>
__global__ void __launch_bounds__(kValueThreads, R == 256 && NT == 16 ? 2 : 1) project_value_kernel(const __grid_constant__ AbsorbedArgs a) {
    using Smem = ValueSmem<R, NT>;
    constexpr int NC = Smem::NC, NW = Smem::NW;
    extern __shared__ __align__(1024) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const Step& m = a.m;
    const int tid = threadIdx.x, warp = warp_id(), lane = tid & 31;
    // (the plan and the step's tables do not come from the kernel before: its CTAs have all begun, so what precedes them is complete)
    const int B = m.num_sequences, count = a.token_prefix[B], tiles = (count + NT - 1) / NT * m.H;
    if ((int)blockIdx.x >= tiles) {
        pa::grid_wait();
        return;
    }
    if (tid == kJoinThreads) {
        for (int i = 0; i < NW; ++i) { pa::mbar_init(&sm.w_full[i], 1); pa::mbar_init(&sm.w_free[i], 1); }
        pa::mbar_init(&sm.o_full, kJoinWarps);
        pa::mbar_init(&sm.done, 1);
        pa::mbar_init(&sm.idle, 1);
        pa::mbar_fence_init();
        sm.abort_flag = 0;
    }
    __syncthreads();
    if (warp == kJoinWarps) tc05::tmem_alloc(&sm.tmem_base, 64);
    const Waiter wt{&sm.abort_flag, m.status, m.wait_polls};
    uint32_t parity = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, parity ^= 1) {
        const int h = tile % m.H, c0 = tile / m.H * NT, rows = min(NT, count - c0);
        if (tid < rows) {      // the tile's tokens: of those of this form the ones from number c0
            const int c = c0 + tid;
            int lo = 0, hi = B;
            if (c < B && a.token_prefix[c] == c && a.token_prefix[c + 1] == c + 1) lo = c;
            else
                while (hi - lo > 1) {        // token_prefix[lo] <= c < token_prefix[hi]
                    const int mid = (lo + hi) >> 1;
                    if (a.token_prefix[mid] <= c) lo = mid; else hi = mid;
                }
            sm.token[tid] = m.subsequence_begins[lo] + c - a.token_prefix[lo];
        }
        auto load_weights = [&](int c) {
            if (tc05::elect_one()) {
                pa::mbar_expect_tx(&sm.w_full[c % NW], m.Dv * 128);
                tma_3d(sm.w[c % NW], &a.map_value_up, c * 64, 0, h, &sm.w_full[c % NW]);
            }
            __syncwarp();
        };
        if (warp == kJoinWarps)
            for (int c = 0; c < NW; ++c) load_weights(c);
        if (tile == (int)blockIdx.x) pa::grid_wait();
        tc05::fence_before_thread_sync();
        __syncthreads();
        tc05::fence_after_thread_sync();
        const uint32_t tmem = sm.tmem_base;
        if (warp == kJoinWarps) {
            bool ok = true;
            const uint32_t idesc = tc05::instr_desc_f16(m.Dv, NT, BF ? 1 : 0, 0, 0), dw = desc_low(sm.w), doh = desc_low(sm.o[0]), dol = desc_low(sm.o[1]);
            constexpr uint32_t kTurns = NC / NW;      // uses of a buffer to a tile
            static_assert(NC % NW == 0, "");
            int loaded = NW;
            ok = wt.wait_warp(&sm.o_full, parity);
            for (int c = 0; ok && c < NC; ++c) {
                ok = wt.wait_warp(&sm.w_full[c % NW], (kTurns * parity + c / NW) & 1);
                if (!ok) break;
                tc05::fence_after_thread_sync();
                const uint32_t da = dw + c % NW * (128 * 128 >> 4), dh = doh + c * (NT * 128 >> 4), dl = dol + c * (NT * 128 >> 4);
                if (tc05::elect_one()) {
                    if (c == 0) mma_ss<0>(tmem, da, dh, idesc);
                    else mma_ss<1>(tmem, da, dh, idesc);
#pragma unroll
                    for (int kk = 1; kk < 4; ++kk) mma_ss<1>(tmem, da + 2 * kk, dh + 2 * kk, idesc);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) mma_ss<1>(tmem, da + 2 * kk, dl + 2 * kk, idesc);
                    tc05::commit(&sm.w_free[c % NW]);
                    if (c + 1 == NC) tc05::commit(&sm.done);
                }
                __syncwarp();
                if (c + NW < NC) {
                    ok = wt.wait_warp(&sm.w_free[c % NW], (kTurns * parity + c / NW) & 1);
                    if (ok) { load_weights(c + NW); ++loaded; }
                }
            }
            if (!ok)
                for (int c = max(0, loaded - NW); c < loaded; ++c) drain(&sm.w_full[c % NW], (kTurns * parity + c / NW) & 1);
        } else {
            const int step = a.row_tiles * kTile;        // from a row's partial result to the next
            auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kJoinThreads) : "memory"); };   // (the joining warps; none of them can have left)
            // element quad `e` of row `r`, swizzled by the row
            auto store = [&](int r, int e, const float (&y)[4]) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    hi[i] = pack2<BF>(y[2 * i], y[2 * i + 1]);
                    lo[i] = pack2<BF>(y[2 * i] - unpack1<BF>((uint16_t)hi[i]), y[2 * i + 1] - unpack1<BF>((uint16_t)(hi[i] >> 16)));
                }
                const uint32_t at = r * 128 + (((e % 16 >> 1) ^ (r & 7)) << 4) + (e & 1) * 8;
                *reinterpret_cast<uint2*>(sm.o[0][e / 16] + at) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(sm.o[1][e / 16] + at) = make_uint2(lo[0], lo[1]);
            };
            // A warp has a row (of 64: one of every sixteen), or rows that are fewer than the warps have several each, which deal out the pieces.
            // A lane has four elements of every 128, and the statistics of one of 32 pieces; the first pieces are under way before their weights are known.
            constexpr int V = R / 128, kRows = NT / kJoinWarps, U = NT == 16 ? 4 : 2;
            const int spread = NT == 16 ? 4 - (32 - __clz(rows - 1)) : 0;
            const int each = 1 << spread, mine = warp & (each - 1);
            int2 part[kRows];
            float2 ml[kRows];
            float4 p[2][U][V];
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int r = (warp >> spread) + u * kJoinWarps;
                part[u] = r < rows ? checked_part(a.row_part[(long long)sm.token[r] * m.H + h], step, a.part_rows) : make_int2(0, 0);
            }
            auto load = [&](float4 (&q)[V], const int2& row, int piece) {
                const float4* src = reinterpret_cast<const float4*>(a.part_o + (row.x + (long long)piece * step) * R) + lane;
#pragma unroll
                for (int v = 0; v < V; ++v) q[v] = src[32 * v];
            };
            auto first = [&](int u) {
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (mine + k * each < part[u].y) load(p[u & 1][k], part[u], mine + k * each);
            };
#pragma unroll
            for (int u = 0; u < kRows; ++u) ml[u] = lane < part[u].y ? a.part_ml[part[u].x + (long long)lane * step] : make_float2(-INFINITY, 0.f);
            first(0);
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int r = (warp >> spread) + u * kJoinWarps, pieces = part[u].y;
                if (u + 1 < kRows) first(u + 1);
                // the pieces' common maximum, and the denominator.  A piece whose tiles the row does not see has a sum of zero and is passed over; one
                // whose logits hold not-a-number or infinity has a sum that is not-a-number, which goes through to the row
                float top = ml[u].y != 0.f ? ml[u].x : -INFINITY, sum = ml[u].y;
                for (int i = lane + 32; i < pieces; i += 32) {
                    const float2 other = a.part_ml[part[u].x + (long long)i * step];
                    if (other.y != 0.f) {
                        const float t = fmaxf(top, other.x);
                        sum = (sum == 0.f ? 0.f : sum * ex2(top - t)) + other.y * ex2(other.x - t);
                        top = t;
                    }
                }
                const float most = pa::warp_max(top), inv = 1.f / pa::warp_sum(sum == 0.f ? 0.f : sum * ex2(top - most));
                float y[V][4];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v][0] = y[v][1] = y[v][2] = y[v][3] = 0.f * inv;      // (not-a-number for a row without any sum, or whose sum is)
                for (int base = 0; base < pieces; base += 32 * each) {
                    const int i = base + mine + lane * each, count = min(32, (pieces - base - mine + each - 1) >> spread);
                    float2 own = ml[u];
                    if (base > 0 || each > 1) own = i < pieces ? a.part_ml[part[u].x + (long long)i * step] : make_float2(-INFINITY, 0.f);
                    const float weight = own.y != 0.f ? ex2(own.x - most) * inv : 0.f;
                    for (int j = 0; j < count; j += U) {
                        if (base + j > 0) {
#pragma unroll
                            for (int k = 0; k < U; ++k)
                                if (j + k < count) load(p[u & 1][k], part[u], base + mine + (j + k) * each);
                        }
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            const float f = __shfl_sync(0xffffffffu, weight, j + k);
                            if (f != 0.f) {      // (a piece without sums has no results either)
#pragma unroll
                                for (int v = 0; v < V; ++v) {
                                    const float4& q = p[u & 1][k][v];
                                    y[v][0] += f * q.x; y[v][1] += f * q.y; y[v][2] += f * q.z; y[v][3] += f * q.w;
                                }
                            }
                        }
                    }
                }
                if (each == 1) {
                    if (pieces > 0) {
#pragma unroll
                        for (int v = 0; v < V; ++v) store(r, lane + 32 * v, y[v]);
                    }
                } else {
                    // the sums of a row's warps, in turn where the rows will be
                    float4* sums = reinterpret_cast<float4*>(sm.o);
                    static_assert(NT != 16 || sizeof(sm.o) == kJoinWarps * R * 4, "");
#pragma unroll
                    for (int v = 0; v < V; ++v) sums[warp * (R / 4) + lane + 32 * v] = make_float4(y[v][0], y[v][1], y[v][2], y[v][3]);
                    meet();
                    float z[2][4] = {};
#pragma unroll
                    for (int x = 0; x < 2; ++x) {      // (at most eight rows)
                        const int unit = tid + x * kJoinThreads;
                        if (unit < rows * (R / 4))
                            for (int k = 0; k < each; ++k) {
                                const float4 q = sums[((unit / (R / 4) << spread) + k) * (R / 4) + unit % (R / 4)];
                                z[x][0] += q.x; z[x][1] += q.y; z[x][2] += q.z; z[x][3] += q.w;
                            }
                    }
                    meet();
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int unit = tid + x * kJoinThreads;
                        if (unit < rows * (R / 4)) store(unit / (R / 4), unit % (R / 4), z[x]);
                    }
                }
            }
            tc05::fence_proxy_async_smem();
            warp_arrive(&sm.o_full);
            if (warp < 4) {
                const bool ok = wt.wait_warp(&sm.done, parity);
                tc05::fence_after_thread_sync();
                // 128 rows: a warp has 32 of them; 64 rows: 16, in the first half of its lanes
                const int d = m.Dv == 128 ? 32 * warp + lane : 16 * warp + lane;
                if (ok) {
                    uint16_t* dst = (uint16_t*)a.output + (long long)h * m.Dv + d;
#pragma unroll
                    for (int g = 0; g < NT; g += 16) {
                        uint32_t r[16];
                        tc05::ld_32x32b_x16(tmem + ((uint32_t)(warp * 32) << 16) + g, r);
                        tc05::wait_ld();
                        if (m.Dv == 128 || lane < 16) {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (g + c < rows) dst[(long long)sm.token[g + c] * m.H * m.Dv] = pack1<BF>(__uint_as_float(r[c]));
                        }
                    }
                }
            }
        }
        tc05::fence_before_thread_sync();
        __syncthreads();
        tc05::fence_after_thread_sync();
        if (*(volatile int*)&sm.abort_flag) break;
    }
    if (warp == kJoinWarps) {
        if (*(volatile int*)&sm.abort_flag) drain_products(&sm.idle);
        tc05::tmem_dealloc(sm.tmem_base, 64);
    }
}

int query_smem(int Dn) { return 2 * Dn * 128 + Dn / 64 * 8192; }

template <int R, bool BF>
cudaError_t launch(const AbsorbedArgs& a, cudaStream_t stream, int* launches) {
    const Step& m = a.m;
    const int token_tiles = (m.num_tokens + kTile - 1) / kTile;
    cudaError_t e = pa::launch_dependent(project_query_kernel<BF>, 1 + token_tiles * m.H * (R / 128), 128, query_smem(m.Dn), stream, a);
    if (e == cudaSuccess) e = pa::launch_dependent(attend_kernel<R, BF>, a.groups * a.row_tiles, kThreads, sizeof(AttendSmem<R>), stream, a);
    if (e == cudaSuccess) {
        // tiles of 16 tokens where those of 64 would leave SMs without one; in an AUTO step most tokens may be the expanded form's
        const int rows = m.form == PA_LATENT_AUTO ? std::min(m.num_tokens, m.num_sequences) : m.num_tokens;
        const int sms = a.groups * a.row_tiles, few = (m.num_tokens + 15) / 16 * m.H, many = token_tiles * m.H;
        if (rows <= 16 || (long long)(rows + kTile - 1) / kTile * m.H < sms * 2 / 3)
            e = pa::launch_dependent(project_value_kernel<R, 16, BF>, std::min(few, R == 256 ? 2 * sms : sms), kValueThreads, sizeof(ValueSmem<R, 16>), stream, a);
        else e = pa::launch_dependent(project_value_kernel<R, 64, BF>, std::min(many, sms), kValueThreads, sizeof(ValueSmem<R, 64>), stream, a);
    }
    *launches += 3;
    return e;
}

template <int R, bool BF>
cudaError_t prepare(const Step& m) {
    // (for the largest size: the kernel serves operators of several, and the limit is the kernel's)
    cudaError_t e = cudaFuncSetAttribute(project_query_kernel<BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, query_smem(128));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_kernel<R, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(AttendSmem<R>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(project_value_kernel<R, 16, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ValueSmem<R, 16>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(project_value_kernel<R, 64, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ValueSmem<R, 64>));
    return e;
}

}  // namespace

long long absorbed_slots(int tokens, int sequences, int heads, int groups, int row_tiles) {
    // a sequence of n tokens has ceil(n * heads / rows) blocks; that is at most n * ceil(heads / rows), and n * heads / rows + 1
    const long long rows = (long long)kTile * row_tiles;
    const long long blocks = std::min(tokens * ((heads + rows - 1) / rows), (long long)tokens * heads / rows + sequences);
    return (blocks + groups) * row_tiles;
}

cudaError_t launch_absorbed(const AbsorbedArgs& a, int dtype, cudaStream_t stream, int* launches) {
    if (dtype == PA_DTYPE_BF16) return a.m.R == 512 ? launch<512, true>(a, stream, launches) : launch<256, true>(a, stream, launches);
    return a.m.R == 512 ? launch<512, false>(a, stream, launches) : launch<256, false>(a, stream, launches);
}

cudaError_t prepare_absorbed(const Step& m, int dtype) {
    if (dtype == PA_DTYPE_BF16) return m.R == 512 ? prepare<512, true>(m) : prepare<256, true>(m);
    return m.R == 512 ? prepare<512, false>(m) : prepare<256, false>(m);
}

}  // namespace latent
