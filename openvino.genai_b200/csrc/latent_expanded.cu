// Latent attention in its expanded form, on the 5th-generation tensor cores (tcgen05 + TMEM): keys and values of the served contexts are
// made per head (k = key_up c, v = value_up c), then attention over them.
//   plan     context tiles and query tiles of the sequences, query tiles longest context first
//   expand   k, v of every (128 context tokens, head), and the rotated key part gathered from its pages
//   attend   256 new tokens of one head at a time
#include <algorithm>
#include <climits>

#include "latent_tc.cuh"

namespace latent {

namespace {

// ---- plan ------------------------------------------------------------------------------------------------------------------
constexpr int kBuckets = 1024;
constexpr int kListed = 1024;       // query tiles that are listed in shared memory; later ones are searched for
__global__ void __launch_bounds__(256) expanded_plan_kernel(const __grid_constant__ ExpandedArgs a) {
    __shared__ int sh_c[8], sh_q[8], run_c, run_q;
    __shared__ int bucket[kBuckets];
    __shared__ int3 listed[kListed];     // sequence, query tile, context tiles
    __shared__ unsigned long long all_c, all_t, work;
    __shared__ int deepest, cuts[32], longest, pieces_sum, slots;
    const Step& m = a.m;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, B = m.num_sequences;
    pa::grid_wait();
    pa::grid_release();
    if (tid == 0) { run_c = 0; run_q = 0; all_c = all_t = work = 0; deepest = pieces_sum = slots = 0; }
    // (every sequence looks at its own slice of the prefix sums; tokens in front of the first and behind the last are nobody's)
    if (tid == 0 && (m.subsequence_begins[0] != 0 || m.subsequence_begins[B] != m.num_tokens)) atomicOr(m.status, PA_DEV_BAD_BEGINS);
    if (tid < 32) cuts[tid] = 0;
    for (int i = tid; i < a.passes; i += 256) a.counter[i] = 0;
    for (int i = tid; i < a.passes * a.part_slots * 8; i += 256) a.arrived[i] = 0;
    for (int i = tid; i < kBuckets; i += 256) bucket[i] = 0;
    __syncthreads();
    for (int base = 0; base < B; base += 256) {
        const int s = base + tid;
        int c = 0, q = 0;
        SeqView v{0, 0, 0, 0};
        if (s < B) {
            if (seq_view(m, s, v) && v.n > 0 && !takes_absorbed(m, v)) {
                c = (int)(((long long)v.past + v.n + kExpandTile - 1) / kExpandTile);
                q = (v.n + kQueryTile - 1) / kQueryTile;
                atomicAdd(&all_c, (unsigned long long)c);
                atomicAdd(&all_t, (unsigned long long)v.n);
                atomicMax(&deepest, c);
            }
        }
        const int mine_c = c, mine_q = q;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int pc = __shfl_up_sync(0xffffffffu, c, o), pq = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) { c += pc; q += pq; }
        }
        if (lane == 31) { sh_c[wid] = c; sh_q[wid] = q; }
        __syncthreads();
        int off_c = run_c, off_q = run_q;
        for (int w = 0; w < wid; ++w) { off_c += sh_c[w]; off_q += sh_q[w]; }
        if (s < B) { a.tile_prefix[s] = off_c + c - mine_c; a.query_prefix[s] = off_q + q - mine_q; }
        unsigned long long sum = 0;
        for (int k = 0; k < mine_q; ++k) {
            const int at = off_q + q - mine_q + k, tiles = (int)(((long long)v.past + min(v.n, (k + 1) * kQueryTile) + kExpandTile - 1) / kExpandTile);
            if (at < kListed) listed[at] = make_int3(s, k, tiles);
            sum += tiles;
        }
        if (mine_q > 0) atomicAdd(&work, sum);
        __syncthreads();
        if (tid == 255) { run_c = off_c + c; run_q = off_q + q; }
        __syncthreads();
    }
    // Prefix sums that fall can give sequences the same tokens or blocks, more in all than the workspace has rows for: such a step gets no plan.
    if (all_t > (unsigned long long)m.num_tokens || all_c * kExpandTile > (unsigned long long)a.rows) {
        if (tid == 0) {
            atomicOr(m.status, PA_DEV_BAD_BEGINS);
            a.tile_prefix[B] = 0;
            *a.heads_per_item = 1;
            *a.items = 0;
        }
        return;
    }
    if (tid == 0) { a.tile_prefix[B] = run_c; a.query_prefix[B] = run_q; }
    if (tid >= 32 && tid < 64) {
        // heads of an item of the expansion: the number whose last CTA ends first, at 7 parts a head and 4 for bringing the context tile in
        const int per = lane + 1;
        const long long items = (long long)run_c * ((a.heads + per - 1) / per);
        long long cost = per <= a.heads ? (items + a.ctas - 1) / a.ctas * (7 * per + 4) : LLONG_MAX / 64;
        cost = cost * 32 + lane;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) cost = min(cost, __shfl_xor_sync(0xffffffffu, cost, o));
        if (lane == 0) *a.heads_per_item = (int)(cost % 32) + 1;
    }
    __syncthreads();
    // Query tiles are cut along their context where they are too few for the CTAs: into the pieces whose rounds over the CTAs end first, at two tiles to a
    // piece for its beginning and end, and three for the joining.  None is shorter than a CTA's share of all tiles, and a cut tile has more than one
    // piece's worth, so that there are at most 2 * ctas pieces of cut ones.  (Three prompts by 16 heads, 96 tiles of 7 to 19 x 128 context tokens, beside 40
    // rows of one token: 146 us uncut, 134 in pieces of at most 10, 151 in pieces of 8, which take a second round.)
    const int total = run_q;
    auto place = [&](int i, int& s, int& qt) {       // context tiles of query tile i
        if (i < kListed) {
            s = listed[i].x;
            qt = listed[i].y;
            return listed[i].z;
        }
        int lo = 0, hi = B;   // query_prefix[lo] <= i < query_prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.query_prefix[mid] <= i) lo = mid; else hi = mid;
        }
        s = lo;
        qt = i - a.query_prefix[lo];
        const int n = m.subsequence_begins[lo + 1] - m.subsequence_begins[lo];
        return (m.past_lens[lo] + min(n, (qt + 1) * kQueryTile) + kExpandTile - 1) / kExpandTile;
    };
    const long long share = ((long long)work * a.heads + a.ctas - 1) / a.ctas;
    const bool few = a.part_slots > 0 && deepest > share && total <= kListed;
    if (few) {
        const int most = max((deepest + lane) / (lane + 1), (int)share);      // a warp for every eighth tile, a lane for every length
        int pieces = 0;
        for (int i = wid; i < total; i += 8) {
            int s, qt;
            pieces += (place(i, s, qt) + most - 1) / most;
        }
        atomicAdd(&cuts[lane], pieces);
        __syncthreads();
        if (tid < 32) {
            const long long rounds = ((long long)cuts[lane] * a.heads + a.ctas - 1) / a.ctas;
            long long cost = (rounds * (most + 2) + (lane > 0 ? 3 : 0)) * 32 + lane;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) cost = min(cost, __shfl_xor_sync(0xffffffffu, cost, o));
            if (lane == cost % 32) longest = most;
        }
    } else if (tid == 0) longest = INT_MAX / 2;
    __syncthreads();
    auto cut = [&](int tiles, int& length) {         // pieces of a query tile, and their length
        const int pieces = (tiles + longest - 1) / longest;
        length = (tiles + pieces - 1) / pieces;
        return (tiles + length - 1) / length;
    };
    // counting sort of the pieces by length, the longest first, so that the last items to be drawn are short
    for (int i = tid; i < total; i += 256) {
        int s, qt, length;
        const int tiles = place(i, s, qt), pieces = cut(tiles, length);
        for (int k = 0; k < pieces; ++k) atomicAdd(&bucket[kBuckets - 1 - min(min(length, tiles - k * length), kBuckets - 1)], 1);
        atomicAdd(&pieces_sum, pieces);
    }
    __syncthreads();
    if (tid < 32) {          // exclusive prefix sum over the buckets
        int run = 0;
        for (int base = 0; base < kBuckets; base += 32) {
            const int mine = bucket[base + lane];
            int v = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int p = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += p;
            }
            bucket[base + lane] = run + v - mine;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    if (tid == 0) *a.items = pieces_sum;
    for (int i = tid; i < total; i += 256) {
        int s, qt, length;
        const int tiles = place(i, s, qt), pieces = cut(tiles, length), slot = pieces > 1 ? atomicAdd(&slots, pieces) : -1;
        for (int k = 0; k < pieces; ++k)
            a.order[atomicAdd(&bucket[kBuckets - 1 - min(min(length, tiles - k * length), kBuckets - 1)], 1)] = PieceOfQuery{s, qt, k, length, slot};
    }
}

// ---- k = key_up c, v = value_up c ---------------------------------------------------------------------------------------------
// A CTA keeps a tile of 128 context rows in tensor memory and walks over heads: D[token][element] of the head's keys, then of its values, with the
// weights streamed in chunks of 64 latent elements.  Keys and values have an accumulator each, so that one is written out while the other is
// computed.  The rows go from the cache to shared memory (the next tile's beside this one's products) and from there to tensor memory, because an
// M 128, N 128 step with both operands in shared memory takes all of that memory's bandwidth and leaves none for the weights to come in:
// 13,143 rows by 32 heads of 512 -> 128 + 128 take 112 us (tensor pipe 49 % busy, 157 MB of the results written back).  A head's tile takes 7000 cycles
// and its products 4096: the weights, which every tile brings in again from the L2 cache, arrive no faster beside them.
// Keys and values are rounded to 16 bits, as operands of the attention's products.
constexpr int kExpandThreads = 224;    // warps 0 - 3: output, 4: rows and even chunks of weights, 5: products, 6: odd chunks (one warp takes 450 cycles a chunk, the products 256)

// A place in a ring of N barriers and the phase that it waits for.
template <int N>
struct Ring {
    uint32_t at = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) { at = 0; phase ^= 1u; }
    }
};

template <int R>
struct ExpandSmem {
    static constexpr int NW = R == 512 ? 5 : 8;              // chunks of weights under way: what the context tile leaves room for
    alignas(1024) uint8_t a[R / 64][kExpandTile * 128];
    alignas(1024) uint8_t w[NW][128 * 128];
    alignas(1024) uint8_t out[kExpandTile * 128];            // 64 elements of every row on their way to global memory
    uint64_t a_full, a_free, a_ready;                        // rows in shared memory, read, in tensor memory
    uint64_t w_full[NW], w_free[NW], d_full[2], d_free[2];   // weights; accumulators of keys and values
    uint64_t idle;                                           // after an abort
    uint32_t asked[3];                                       // the loaders' last words: context tiles, chunks of weights up to each one's last
    uint32_t tmem_base;
    int abort_flag;
};

struct ExpandItem {
    int s, tile, h_first, h_end;    // sequence, its context tile, heads (of this pass)
    int valid;                      // rows of the tile inside the context
    int row;                        // first row in the scratch
    int block0, blocks;             // its blocks inside block_indices
};

__device__ __forceinline__ ExpandItem expand_item(const ExpandedArgs& a, int i, int per) {
    const int head_groups = (a.heads + per - 1) / per, tile = i / head_groups;
    ExpandItem it;
    it.h_first = i % head_groups * per;
    it.h_end = min(a.heads, it.h_first + per);
    int lo = 0, hi = a.m.num_sequences;   // tile_prefix[lo] <= tile < tile_prefix[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.tile_prefix[mid] <= tile) lo = mid; else hi = mid;
    }
    it.s = lo;
    it.tile = tile - a.tile_prefix[lo];
    SeqView v;
    seq_view(a.m, lo, v);
    const int from = it.tile * kExpandTile;
    it.valid = min(kExpandTile, v.past + v.n - from);
    it.row = tile * kExpandTile;
    it.block0 = v.tb + from / a.m.bs;
    it.blocks = (it.valid + a.m.bs - 1) / a.m.bs;
    return it;
}

template <int R, int DN, int DV, bool BF>
__global__ void __launch_bounds__(kExpandThreads, 1) expand_kernel(const __grid_constant__ ExpandedArgs a) {
    using Smem = ExpandSmem<R>;
    constexpr int NC = R / 64, NW = Smem::NW;
    extern __shared__ __align__(1024) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const Step& m = a.m;
    const int tid = threadIdx.x, warp = warp_id(), lane = tid & 31;
    if (tid == 0) {
        pa::mbar_init(&sm.a_full, 1);
        pa::mbar_init(&sm.a_free, 4);
        pa::mbar_init(&sm.a_ready, 4);
        pa::mbar_init(&sm.idle, 1);
        for (int i = 0; i < NW; ++i) { pa::mbar_init(&sm.w_full[i], 1); pa::mbar_init(&sm.w_free[i], 1); }
        for (int i = 0; i < 2; ++i) { pa::mbar_init(&sm.d_full[i], 1); pa::mbar_init(&sm.d_free[i], 4); }
        pa::mbar_fence_init();
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
    const int per = min(*a.heads_per_item, a.heads), items = a.tile_prefix[m.num_sequences] * ((a.heads + per - 1) / per);
    constexpr uint32_t kD = R / 2;       // tensor memory: the rows (two elements a column), then 128 columns each for keys and values

    if (warp == 4 || warp == 6) {
        const bool even = warp == 4;
        uint32_t n = 0, tiles = 0, chunks = 0;
        bool ok = true, bad_index = false;
        for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
            const ExpandItem it = expand_item(a, i, per);
            if (even) {
                int page = 0;
                if (lane < it.blocks) {
                    page = m.block_indices[it.block0 + lane];
                    if (page < 0 || page >= m.num_blocks) { page = 0; bad_index = true; }
                }
                if (tiles > 0) ok = wt.wait_warp(&sm.a_free, (tiles - 1) & 1);
                if (!ok) break;
                ++tiles;
                if (tc05::elect_one()) pa::mbar_expect_tx(&sm.a_full, it.blocks * m.bs * 128 * NC);
                __syncwarp();
                for (int b = 0; b < it.blocks; ++b) {
                    const int at = __shfl_sync(0xffffffffu, page, b) * m.bs;
                    if (tc05::elect_one())
                        for (int c = 0; c < NC; ++c) tma_2d(sm.a[c] + b * m.bs * 128, &a.map_cache, 64 * c, at, &sm.a_full);
                    __syncwarp();
                }
            }
            for (int h = it.h_first; ok && h < it.h_end; ++h)
                for (int x = 0; ok && x < 2 * NC; ++x, ++n) {
                    if ((n & 1) == (even ? 1u : 0u)) continue;
                    const int st = n % NW;
                    if (n >= NW) ok = wt.spin_warp(&sm.w_free[st], (n / NW - 1) & 1);
                    if (ok && tc05::elect_one()) {
                        pa::mbar_expect_tx(&sm.w_full[st], (x < NC ? DN : DV) * 128);
                        tma_3d(sm.w[st], x < NC ? &a.map_key_up : &a.map_value_up, 64 * (x % NC), 0, a.h0 + h, &sm.w_full[st]);
                    }
                    __syncwarp();
                    if (ok) chunks = n + 1;
                }
        }
        if (__any_sync(0xffffffffu, bad_index) && lane == 0) atomicOr(m.status, PA_DEV_BAD_BLOCK_INDEX);
        if (lane == 0) {
            if (even) sm.asked[0] = tiles;
            sm.asked[even ? 1 : 2] = chunks;
        }
    } else if (warp == 5) {
        constexpr uint32_t idesc_k = tc05::instr_desc_f16(128, DN, BF ? 1 : 0, 0, 0), idesc_v = tc05::instr_desc_f16(128, DV, BF ? 1 : 0, 0, 0);
        Ring<NW> w;
        const uint32_t dw = desc_low(sm.w);
        uint32_t na = 0, nd = 0;
        bool ok = true;
        for (int i = blockIdx.x; ok && i < items; i += gridDim.x, ++na) {
            const ExpandItem it = expand_item(a, i, per);
            ok = wt.spin_warp(&sm.a_ready, na & 1);
            for (int h = it.h_first; ok && h < it.h_end; ++h, ++nd)
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    if (ok && nd > 0) ok = wt.spin_warp(&sm.d_free[part], (nd - 1) & 1);
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        if (ok) ok = wt.spin_warp(&sm.w_full[w.at], w.phase);
                        if (!ok) break;
                        tc05::fence_after_thread_sync();
                        const uint32_t d = tmem + kD + part * 128, rows = tmem + c * 32, pw = dw + w.at * (128 * 128 >> 4), idesc = part ? idesc_v : idesc_k;
                        if (tc05::elect_one()) {
                            if (c == 0) mma_ts<0>(d, rows, pw, idesc);
                            else mma_ts<1>(d, rows, pw, idesc);
#pragma unroll
                            for (int kk = 1; kk < 4; ++kk) mma_ts<1>(d, rows + 8 * kk, pw + 2 * kk, idesc);
                            tc05::commit(&sm.w_free[w.at]);
                            if (c + 1 == NC) tc05::commit(&sm.d_full[part]);
                        }
                        __syncwarp();
                        w.next();
                    }
                }
        }
    } else {
        uint32_t nd = 0, na = 0;
        const int row = tid;       // of the tile
        const bool leader = tc05::elect_one();     // the lane whose copies and waits for them are the warp's
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        // this thread's row from shared to tensor memory
        auto keep_rows = [&]() -> bool {
            if (!wt.wait_warp(&sm.a_full, na & 1)) return false;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t r[32];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint4 v = *reinterpret_cast<const uint4*>(sm.a[c] + row * 128 + ((q ^ (row & 7)) << 4));
                    r[4 * q] = v.x; r[4 * q + 1] = v.y; r[4 * q + 2] = v.z; r[4 * q + 3] = v.w;
                }
                tc05::st_32x32b_x32(tmem + c * 32 + lanes, r);
            }
            tc05::wait_st();
            tc05::fence_before_thread_sync();
            warp_arrive(&sm.a_ready);
            warp_arrive(&sm.a_free);
            ++na;
            return true;
        };
        bool ok = true;
        if ((int)blockIdx.x < items) ok = keep_rows();
        for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
            const ExpandItem it = expand_item(a, i, per);
            const bool live = row < it.valid;
            if (it.h_first == 0 && a.h0 == 0) {      // the rotated part of the keys, once
                uint4* dst = reinterpret_cast<uint4*>((uint16_t*)a.k_rope + ((long long)it.row + row) * 64);
                const uint4* src = nullptr;
                if (live) {
                    const int page = m.block_indices[it.block0 + row / m.bs];
                    if (page >= 0 && page < m.num_blocks)
                        src = reinterpret_cast<const uint4*>((const uint16_t*)a.cache + ((long long)page * m.bs + row % m.bs) * (m.R + m.P) + m.R);
                }
                for (int c = 0; c < m.P / 8; ++c) dst[c] = src ? src[c] : make_uint4(0, 0, 0, 0);
            }
            for (int h = it.h_first; ok && h < it.h_end; ++h, ++nd) {
                // 64 elements of the warp's 32 rows at a time
#pragma unroll
                for (int c0 = 0; c0 < DN + DV; c0 += 64) {
                    const bool value = c0 >= DN;
                    const int at = value ? c0 - DN : c0, size = value ? DV : DN;
                    if (at == 0) {
                        if (ok) ok = wt.wait_warp(&sm.d_full[value], nd & 1);
                        if (!ok) break;
                        tc05::fence_after_thread_sync();
                        // (the item's last product is complete: the next item's rows may take the place of this one's)
                        if (value && h + 1 == it.h_end && i + (int)gridDim.x < items) ok = keep_rows();
                        if (!ok) break;
                    }
                    const uint32_t src = tmem + kD + (value ? 128 : 0) + at + lanes;
                    uint32_t r[2][32];
                    tc05::ld_32x32b_x32(src, r[0]);
                    tc05::ld_32x32b_x32(src + 32, r[1]);
                    tc05::wait_ld();
                    if (at + 64 == size) {
                        tc05::fence_before_thread_sync();
                        warp_arrive(&sm.d_free[value]);
                    }
                    // the copy out of the warp's staging rows before has read them
                    if (leader) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const uint32_t* v = &r[q >> 2][8 * (q & 3)];
                        uint4 w = make_uint4(0, 0, 0, 0);     // rows behind the context: zeros, whatever the cache holds there
                        if (live)
                            w = make_uint4(pack2<BF>(__uint_as_float(v[0]), __uint_as_float(v[1])), pack2<BF>(__uint_as_float(v[2]), __uint_as_float(v[3])),
                                           pack2<BF>(__uint_as_float(v[4]), __uint_as_float(v[5])), pack2<BF>(__uint_as_float(v[6]), __uint_as_float(v[7])));
                        *reinterpret_cast<uint4*>(sm.out + row * 128 + ((q ^ (row & 7)) << 4)) = w;
                    }
                    tc05::fence_proxy_async_smem();
                    __syncwarp();
                    if (leader) {
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(value ? &a.map_v_out : &a.map_k_out),
                                     "r"(at), "r"((int)(h * a.rows + it.row + warp * 32)), "r"(pa::smem_u32(sm.out + warp * 32 * 128)) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    __syncwarp();
                }
            }
        }
        if (leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    __syncthreads();
    if (*(volatile int*)&sm.abort_flag) {
        if (warp == 4 || warp == 6) {
            const uint32_t tiles = sm.asked[0], chunks = sm.asked[warp == 4 ? 1 : 2];
            if (warp == 4 && tiles > 0) drain(&sm.a_full, (tiles - 1) & 1);
            for (uint32_t i = chunks > NW ? chunks - NW : 0; i < chunks; ++i)      // (every other one is this warp's)
                if ((i & 1) == (warp == 6 ? 1u : 0u)) drain(&sm.w_full[i % NW], (i / NW) & 1);
        } else if (warp == 5) drain_products(&sm.idle);
        __syncthreads();
    }
    if (warp == 5) tc05::tmem_dealloc(tmem, 512);
}

// ---- attention ------------------------------------------------------------------------------------------------------------------
// A work item is 256 new tokens of one head in two halves A and B of 128 rows.  S_X = Q_X K^T (M 128, N 128) into TMEM, P_X over S_X, O_X += P_X V
// with P read from TMEM; the tensor core computes P V and the next S of one half beside the softmax of the other.
// Warps 0 - 3 and 4 - 7: softmax of A and B, a thread per row; 8: queries and keys, 9: products, 10: values;
// 11 fills the warpgroup whose registers go to the softmax.
// P is rounded to 16 bits because P and V are one type to the tensor core; S, maxima, sums and O are 32 bits, O is divided once.
// 4 prompts of 1313 - 1891 tokens over 1280 - 1936 by 32 heads (334 GFLOP): 325 us, 1030 TFLOP/s, tensor pipe 53 % busy.  A context tile of both
// halves takes 3850 cycles and its products 2560.  A half's chain is softmax 1840 (maximum 380, 650 for the exponentials of 64 tokens, which is their
// unit's rate) and products 1470, and S may not be overwritten before P is read: O, S and P of both halves fill the tensor memory.  Slower, by the call:
// a third of the exponentials by polynomials (+2 %), the maximum beside the exponentials of a stale one (+1 %), one wait for keys, values and
// P (+3 %), a warp for each half's products (+9 %).
constexpr int kAttendThreads = 384;
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;   // 256 and 128 threads of the 384 x 168 that the CTA is launched with
constexpr int kItemSlots = 4;
constexpr float kGrow = 4.f;       // log2 of the growth of a row maximum that rescales O

struct QueryItem {
    int h;               // head of this pass, -1: no more items
    int t0;              // first new token of the item
    int rows;            // its new tokens
    int past;            // context its first row sees, less one
    int row;             // first row of the sequence's context in the scratch
    int tiles[2];        // context tiles of each half
    int slot, piece;     // partial result of the first piece, -1: the whole context; number of the piece
    int pieces[2];       // of each half
};

template <int DN, int DV>
struct ExpandedSmem {
    static constexpr int NQ = DN / 64 + 1, NV = DV / 64;
    // Rings of key atoms (128 tokens x 64 elements, NQ of them a tile) and of value units (64 tokens): each is freed by itself, so that a
    // tile and a part of the next fit beside the queries
    static constexpr int KS = DN == 128 ? 5 : 4, VS = DN == 128 && DV == 128 ? 3 : DV == 128 ? 4 : 6;
    // One barrier says that all of a tile is there.  There are as many as tiles can have begun to arrive: a loader that came back to one whose tile
    // is still under way would count into the wrong phase.
    static constexpr int TK = (KS + NQ - 1) / NQ, TV = (VS + 1) / 2;
    static_assert(TK == 2, "the loader and the products take turns between two barriers");
    alignas(1024) uint8_t q[2][NQ][128 * 128];
    alignas(1024) uint8_t k[KS][kExpandTile * 128];
    alignas(1024) uint8_t v[VS][NV][64 * 128];
    uint64_t q_full[2], q_free[2], k_full[TK], k_free[KS], v_full[TV], v_free[VS];
    uint64_t s_full[2], p_full[2][2], o_done[2];
    uint64_t idle;             // after an abort
    uint32_t asked[4];         // the loaders' last words: query tiles of both halves, key atoms, value units that they have asked for
    uint64_t item_full[kItemSlots], item_free[kItemSlots];
    QueryItem item[kItemSlots];
    uint32_t tmem_base;
    int abort_flag;
};

template <int N> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int DN, int DV, bool BF>
__global__ void __launch_bounds__(kAttendThreads, 1) expanded_attend_kernel(const __grid_constant__ ExpandedArgs a) {
    using Smem = ExpandedSmem<DN, DV>;
    constexpr int NQ = Smem::NQ, NV = Smem::NV, KS = Smem::KS, VS = Smem::VS, TV = Smem::TV;
    constexpr uint32_t kO = 256;       // S_A, S_B: 128 columns each (P in the first 64), then O_A, O_B
    extern __shared__ __align__(1024) uint8_t smem[];
    Smem& sm = *reinterpret_cast<Smem*>(smem);
    const Step& m = a.m;
    const int tid = threadIdx.x, warp = warp_id(), lane = tid & 31;
    if (tid == 0) {
        for (int x = 0; x < 2; ++x) {
            pa::mbar_init(&sm.q_full[x], 1);
            pa::mbar_init(&sm.k_full[x], 1);
            pa::mbar_init(&sm.q_free[x], 1);
            pa::mbar_init(&sm.s_full[x], 1);
            pa::mbar_init(&sm.p_full[x][0], 4);
            pa::mbar_init(&sm.p_full[x][1], 4);
            pa::mbar_init(&sm.o_done[x], 1);
        }
        pa::mbar_init(&sm.idle, 1);
        for (int i = 0; i < KS; ++i) pa::mbar_init(&sm.k_free[i], 1);
        for (int i = 0; i < VS; ++i) pa::mbar_init(&sm.v_free[i], 1);
        for (int i = 0; i < TV; ++i) pa::mbar_init(&sm.v_full[i], 1);
        for (int i = 0; i < kItemSlots; ++i) { pa::mbar_init(&sm.item_full[i], 1); pa::mbar_init(&sm.item_free[i], 10); }
        pa::mbar_fence_init();
        sm.abort_flag = 0;
    }
    if (warp == 9) tc05::tmem_alloc(&sm.tmem_base, 512);
    tc05::fence_before_thread_sync();
    __syncthreads();
    tc05::fence_after_thread_sync();
    const uint32_t tmem = sm.tmem_base;
    const Waiter wt{&sm.abort_flag, m.status, m.wait_polls};
    auto fetch = [&](uint32_t n, QueryItem& it) -> bool {
        const int slot = n % kItemSlots;
        if (!wt.wait_warp(&sm.item_full[slot], (n / kItemSlots) & 1)) return false;
        it = sm.item[slot];
        warp_arrive(&sm.item_free[slot]);
        return true;
    };

    if (warp >= 8) {
        reg_dec<kOtherRegs>();
        if (warp == 8) {
            // ======================= loader =============================================================
            const int items = *a.items * a.heads;
            uint32_t ni = 0, nk = 0, nq[2] = {0, 0};
            bool ok = true;
            while (ok) {
                int i = blockIdx.x;              // the first item goes by the CTA's number, later ones by turn
                if (ni > 0) {
                    if (lane == 0) i = gridDim.x + atomicAdd(a.counter + a.pass, 1);
                    i = __shfl_sync(0xffffffffu, i, 0);
                }
                QueryItem it;
                it.h = -1;
                if (i < items) {
                    const PieceOfQuery at = a.order[i / a.heads];
                    SeqView v;
                    seq_view(m, at.s, v);
                    const int first = at.piece * at.length, past = v.past + at.tile * kQueryTile;
                    it.h = i % a.heads;
                    it.t0 = v.t0 + at.tile * kQueryTile;
                    it.rows = min(kQueryTile, v.n - at.tile * kQueryTile);
                    it.past = past - first * kExpandTile;
                    it.row = (a.tile_prefix[at.s] + first) * kExpandTile;
                    it.slot = at.slot < 0 ? -1 : at.slot * a.heads + it.h;
                    it.piece = at.piece;
                    for (int x = 0; x < 2; ++x) {
                        const int last = min(it.rows, 128 * (x + 1));     // rows up to the half's end
                        const int tiles = last > 128 * x ? (past + last + kExpandTile - 1) / kExpandTile : 0;
                        it.tiles[x] = min(max(tiles - first, 0), at.length);
                        it.pieces[x] = (tiles + at.length - 1) / at.length;
                    }
                }
                // (the plan and the step's tables do not come from the kernel before, whose CTAs have all begun; keys and values do)
                if (ni == 0) pa::grid_wait();
                const int slot = ni % kItemSlots;
                if (ni >= kItemSlots) ok = wt.wait_warp(&sm.item_free[slot], (ni / kItemSlots - 1) & 1);
                if (!ok) break;
                if (lane == 0) sm.item[slot] = it;
                warp_arrive(&sm.item_full[slot]);
                ++ni;
                if (it.h < 0) break;
                const int tiles = max(it.tiles[0], it.tiles[1]);
                for (int x = 0; ok && x < 2; ++x) {
                    if (it.tiles[x] == 0) continue;
                    if (nq[x] > 0) ok = wt.wait_warp(&sm.q_free[x], (nq[x] - 1) & 1);
                    if (ok && tc05::elect_one()) {
                        pa::mbar_expect_tx(&sm.q_full[x], NQ * 128 * 128);
                        for (int c = 0; c < NQ - 1; ++c) tma_3d(sm.q[x][c], &a.map_qn, 64 * c, a.h0 + it.h, it.t0 + 128 * x, &sm.q_full[x]);
                        tma_3d(sm.q[x][NQ - 1], &a.map_qr, 0, a.h0 + it.h, it.t0 + 128 * x, &sm.q_full[x]);
                    }
                    __syncwarp();
                    nq[x] += ok;
                }
                const int y0 = (int)(it.h * a.rows) + it.row;
                auto load_k = [&](int j) {
                    uint64_t* full = &sm.k_full[nk / NQ & 1];
                    for (int c = 0; ok && c < NQ; ++c, ++nk) {
                        const int st = nk % KS;
                        if (nk >= KS) ok = wt.wait_warp(&sm.k_free[st], (nk / KS - 1) & 1);
                        if (!ok) return;
                        if (tc05::elect_one()) {
                            if (c == 0) pa::mbar_expect_tx(full, NQ * kExpandTile * 128);
                            if (c + 1 < NQ) tma_2d(sm.k[st], &a.map_k, 64 * c, y0 + j * kExpandTile, full);
                            else tma_2d(sm.k[st], &a.map_k_rope, 0, it.row + j * kExpandTile, full);
                        }
                        __syncwarp();
                    }
                };
                for (int j = 0; ok && j < tiles; ++j) load_k(j);
            }
            if (lane == 0) { sm.asked[0] = nq[0]; sm.asked[1] = nq[1]; sm.asked[2] = nk; }
        } else if (warp == 10) {
            // ======================= loader of the values ====================================================
            pa::grid_wait();
            uint32_t nv = 0;
            bool ok = true;
            QueryItem it;
            for (uint32_t ni = 0; ok; ++ni) {
                if (!fetch(ni, it) || it.h < 0) break;
                const int units = 2 * max(it.tiles[0], it.tiles[1]), y0 = (int)(it.h * a.rows) + it.row;
                for (int u = 0; ok && u < units; ++u, ++nv) {
                    const int st = nv % VS;
                    if (nv >= VS) ok = wt.wait_warp(&sm.v_free[st], (nv / VS - 1) & 1);
                    if (!ok) break;
                    uint64_t* full = &sm.v_full[nv / 2 % TV];
                    if (tc05::elect_one()) {
                        if ((u & 1) == 0) pa::mbar_expect_tx(full, 2 * NV * 64 * 128);
                        for (int c = 0; c < NV; ++c) tma_2d(sm.v[st][c], &a.map_v, 64 * c, y0 + 64 * u, full);
                    }
                    __syncwarp();
                }
            }
            if (lane == 0) sm.asked[3] = nv;
        } else if (warp == 9) {
            // ======================= products ============================================================
            // The whole warp runs the loop and one elected lane issues: in code that a single lane runs, an instruction took 110 cycles to issue in
            // place of 50.
            {
                constexpr uint32_t idesc_s = tc05::instr_desc_f16(128, kExpandTile, BF ? 1 : 0, 0, 0);
                constexpr uint32_t idesc_o = tc05::instr_desc_f16(128, DV, BF ? 1 : 0, 0, 1);
                const uint32_t dq = desc_low(sm.q), dk = desc_low(sm.k), dv = desc_low(sm.v, 64 * 128);
                constexpr uint32_t kAtom = 128 * 128 >> 4, kUnit = NV * 64 * 128 >> 4;
                const bool wide = m.P == 64;
                Ring<KS> k[2];           // where each half is in the rings
                Ring<VS> v[2];
                uint32_t nt = 0, nq[2] = {0, 0}, np[2] = {0, 0};     // context tiles before this item; query tiles, P tiles so far
                bool ok = true;
                QueryItem it;
                for (uint32_t ni = 0; ok; ++ni) {
                    if (!fetch(ni, it) || it.h < 0) break;
                    const int tiles = max(it.tiles[0], it.tiles[1]);
                    const int last_half = it.tiles[1] > 0 ? 1 : 0;      // B sees no fewer tiles than A, where it has rows
                    // S of tile j (whose keys are there), by the elected lane
                    auto issue_s = [&](int X, int j) {
                        const uint32_t d = tmem + X * 128;
                        Ring<KS> at = k[X];
#pragma unroll
                        for (int c = 0; c < NQ; ++c, at.next()) {
                            const uint32_t da = dq + (X * NQ + c) * kAtom, db = dk + at.at * kAtom;
                            if (c == 0) mma_ss<0>(d, da, db, idesc_s);
                            else mma_ss<1>(d, da, db, idesc_s);
                            mma_ss<1>(d, da + 2, db + 2, idesc_s);
                            if (c + 1 < NQ || wide) {
                                mma_ss<1>(d, da + 4, db + 4, idesc_s);
                                mma_ss<1>(d, da + 6, db + 6, idesc_s);
                            }
                            if (X == last_half) tc05::commit(&sm.k_free[at.at]);
                        }
                        tc05::commit(&sm.s_full[X]);
                        if (j + 1 == it.tiles[X]) tc05::commit(&sm.q_free[X]);
                    };
                    auto past_keys = [&](int X) {
#pragma unroll
                        for (int c = 0; c < NQ; ++c) k[X].next();
                    };
#pragma unroll
                    for (int X = 0; X < 2; ++X)
                        if (ok && it.tiles[X] > 0) {
                            ok = wt.spin_warp(&sm.q_full[X], nq[X] & 1) && wt.spin_warp(&sm.k_full[nt & 1], (nt >> 1) & 1);
                            ++nq[X];
                            tc05::fence_after_thread_sync();
                            if (ok && tc05::elect_one()) issue_s(X, 0);
                            __syncwarp();
                            past_keys(X);
                        }
                    for (int j = 0; ok && j < tiles; ++j) {
#pragma unroll
                        for (int X = 0; X < 2; ++X)
                            if (ok && j < it.tiles[X]) {
                                // what the loaders bring is waited for first (by A for B too, where both see the tile); the probabilities come later, and
                                // nothing stands between them and their products
                                const bool more = j + 1 < it.tiles[X];
                                const uint32_t n = nt + j;
                                if (X == 0 || j >= it.tiles[0]) ok = wt.spin_warp(&sm.v_full[n % TV], (n / TV) & 1);
                                if (ok && more && (X == 0 || j + 1 >= it.tiles[0])) ok = wt.spin_warp(&sm.k_full[(n + 1) & 1], ((n + 1) >> 1) & 1);
                                const uint32_t d = tmem + kO + X * DV, p = tmem + X * 128;
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    if (ok) ok = wt.spin_warp(&sm.p_full[X][u], np[X] & 1);
                                    if (!ok) break;
                                    tc05::fence_after_thread_sync();
                                    const uint32_t db = dv + v[X].at * kUnit;
                                    if (tc05::elect_one()) {
                                        if (u == 0 && j == 0) mma_ts<0>(d, p + u * 32, db, idesc_o);
                                        else mma_ts<1>(d, p + u * 32, db, idesc_o);
#pragma unroll
                                        for (int kk = 1; kk < 4; ++kk) mma_ts<1>(d, p + u * 32 + kk * 8, db + kk * 128, idesc_o);
                                        if (X == last_half) tc05::commit(&sm.v_free[v[X].at]);
                                        if (u == 1) {
                                            if (more) issue_s(X, j + 1);
                                            else tc05::commit(&sm.o_done[X]);
                                        }
                                    }
                                    __syncwarp();
                                    v[X].next();
                                }
                                ++np[X];
                                if (more) past_keys(X);
                            }
                    }
#pragma unroll
                    for (int X = 0; X < 2; ++X)      // past the tiles that only the other half sees
                        for (int j = it.tiles[X]; j < tiles; ++j) {
                            past_keys(X);
                            v[X].next();
                            v[X].next();
                        }
                    nt += tiles;
                }
            }
        }
    } else {
        // ======================= softmax and output of half X ============================================
        reg_inc<kSoftmaxRegs>();
        const int X = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + X * 128 + lanes, tmem_o = tmem + kO + X * DV + lanes;
        const float c2 = a.scale_log2;
        uint32_t n = 0, no = 0;
        QueryItem it;
        for (uint32_t ni = 0;; ++ni) {
            if (!fetch(ni, it) || it.h < 0) break;
            const int tiles = it.tiles[X];
            if (tiles == 0) continue;
            const int i = 128 * X + r;                      // row of the item
            const int limit = i < it.rows ? it.past + i + 1 : 0;
            const int least = __reduce_min_sync(0xffffffffu, limit);
            float top = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < tiles; ++j, ++n) {
                if (!wt.spin_warp(&sm.s_full[X], n & 1)) { ok = false; break; }
                tc05::fence_after_thread_sync();
                uint32_t s[4][32];
#pragma unroll
                for (int q = 0; q < 4; ++q) tc05::ld_32x32b_x32(tmem_s + 32 * q, s[q]);
                tc05::wait_ld();
                const int seen = limit - j * kExpandTile;
                if ((j + 1) * kExpandTile > least) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (32 * q + c >= seen) s[q][c] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mx[q] = __uint_as_float(s[q][0]);
#pragma unroll
                    for (int c = 1; c < 31; c += 2) mx[q] = max3(mx[q], __uint_as_float(s[q][c]), __uint_as_float(s[q][c + 1]));
                    mx[q] = fmaxf(mx[q], __uint_as_float(s[q][31]));
                }
                const float t = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2;
                float alpha = 1.f;
                bool grew = false;
                if (top == -INFINITY) top = t;
                else if (t > top + kGrow) { alpha = ex2(top - t); top = t; grew = true; }
                if (__any_sync(0xffffffffu, grew)) {     // (the products of the tile before are complete: they precede this tile's S)
#pragma unroll 1
                    for (int q = 0; q < DV / 32; ++q) {
                        uint32_t o[32];
                        tc05::ld_32x32b_x32(tmem_o + 32 * q, o);
                        tc05::wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                        tc05::st_32x32b_x32(tmem_o + 32 * q, o);
                    }
                    l *= alpha;
                }
                const float ref = top == -INFINITY ? 0.f : -top;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                    uint32_t p[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        float x, y;
                        fma2(x, y, __uint_as_float(s[q + (c >> 5)][c & 31]), __uint_as_float(s[q + (c >> 5)][(c & 31) + 1]), c2, ref);
                        x = ex2(x);
                        y = ex2(y);
                        add2(sum[c & 2], sum[(c & 2) + 1], x, y);
                        p[c >> 1] = pack2<BF>(x, y);
                    }
                    tc05::st_32x32b_x32(tmem_s + 16 * q, p);
                    tc05::wait_st();
                    tc05::fence_before_thread_sync();
                    warp_arrive(&sm.p_full[X][q / 2]);      // the products of these 64 tokens run beside the exponentials of the others
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (!ok || !wt.wait_warp(&sm.o_done[X], no & 1)) break;
            ++no;
            tc05::fence_after_thread_sync();
            uint4* dst = reinterpret_cast<uint4*>((uint16_t*)a.output + ((long long)(it.t0 + i) * m.H + a.h0 + it.h) * DV);
            auto put = [&](int q, const uint32_t (&o)[32], float factor) {
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pack2<BF>(__uint_as_float(o[c + 2 * e]) * factor, __uint_as_float(o[c + 2 * e + 1]) * factor);
                    dst[4 * q + c / 8] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            };
            // of a cut context: rows of sums, four elements of 256 rows together
            float4* part = reinterpret_cast<float4*>(a.part_o) + (long long)(it.slot + it.piece * a.heads) * (DV / 4) * kQueryTile + i;
#pragma unroll 1
            for (int q = 0; q < DV / 32; ++q) {
                uint32_t o[32];
                tc05::ld_32x32b_x32(tmem_o + 32 * q, o);
                tc05::wait_ld();
                if (i < it.rows) {
                    if (it.slot < 0) put(q, o, 1.f / l);
                    else
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            part[(8 * q + c / 4) * kQueryTile] = make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
                }
            }
            if (it.slot >= 0) {
                // The warp that is the last of its rows' pieces joins them, in the pieces' order.
                if (i < it.rows) a.part_ml[(long long)(it.slot + it.piece * a.heads) * kQueryTile + i] = make_float2(top, l);
                __threadfence();
                __syncwarp();
                int before = 0;
                if (lane == 0) before = atomicAdd(a.arrived + ((long long)a.pass * a.part_slots + it.slot) * 8 + warp, 1);
                if (__shfl_sync(0xffffffffu, before, 0) + 1 == it.pieces[X]) {
                    __threadfence();
                    if (i < it.rows) {
                        const float2* ml = a.part_ml + (long long)it.slot * kQueryTile + i;
                        const long long step = (long long)a.heads * kQueryTile;
                        float most = -INFINITY, sum = 0.f;
                        for (int k = 0; k < it.pieces[X]; ++k) {
                            const float2 x = __ldcg(ml + k * step);
                            if (x.y == 0.f) continue;       // (a piece that the row does not see)
                            const float to = fmaxf(most, x.x);
                            sum = (sum == 0.f ? 0.f : sum * ex2(most - to)) + x.y * ex2(x.x - to);
                            most = to;
                        }
                        part = reinterpret_cast<float4*>(a.part_o) + (long long)it.slot * (DV / 4) * kQueryTile + i;
#pragma unroll 1
                        for (int q = 0; q < DV / 32; q += 2) {
                            float y[2][32] = {};
#pragma unroll 2
                            for (int k = 0; k < it.pieces[X]; ++k) {
                                const float2 x = __ldcg(ml + k * step);
                                const float f = x.y == 0.f ? 0.f : ex2(x.x - most);
#pragma unroll
                                for (int c = 0; c < 64; c += 4) {
                                    const float4 z = __ldcg(part + k * step * (DV / 4) + (8 * q + c / 4) * kQueryTile);
                                    float* to = &y[c >> 5][c & 31];
                                    to[0] += f * z.x; to[1] += f * z.y; to[2] += f * z.z; to[3] += f * z.w;
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                uint32_t o[32];
#pragma unroll
                                for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(y[e][c]);
                                put(q + e, o, 1.f / sum);
                            }
                        }
                    }
                }
            }
            tc05::fence_before_thread_sync();
        }
    }
    __syncthreads();
    if (*(volatile int*)&sm.abort_flag) {
        // (of a tile that has only begun to be asked for, the rest never comes: that wait ends by the time that a copy can take)
        if (warp == 8) {
            for (int x = 0; x < 2; ++x)
                if (sm.asked[x] > 0) drain(&sm.q_full[x], (sm.asked[x] - 1) & 1);
            const uint32_t n = (sm.asked[2] + NQ - 1) / NQ;
            for (uint32_t i = n > 2 ? n - 2 : 0; i < n; ++i) drain(&sm.k_full[i & 1], (i >> 1) & 1);
        } else if (warp == 10) {
            const uint32_t n = (sm.asked[3] + 1) / 2;
            for (uint32_t i = n > TV ? n - TV : 0; i < n; ++i) drain(&sm.v_full[i % TV], (i / TV) & 1);
        } else if (warp == 9) drain_products(&sm.idle);
        __syncthreads();
    }
    if (warp == 9) tc05::tmem_dealloc(tmem, 512);
}

template <int R, int DN, int DV, bool BF>
cudaError_t expand_and_attend(const ExpandedArgs& a, int sm_count, cudaStream_t stream, int* launches) {
    cudaError_t e = pa::launch_dependent(expand_kernel<R, DN, DV, BF>, sm_count, kExpandThreads, sizeof(ExpandSmem<R>), stream, a);
    if (e == cudaSuccess) e = pa::launch_dependent(expanded_attend_kernel<DN, DV, BF>, sm_count, kAttendThreads, sizeof(ExpandedSmem<DN, DV>), stream, a);
    *launches += 2;
    return e;
}

template <int R, int DN, int DV, bool BF>
cudaError_t prepare() {
    // the warpgroups re-divide the registers that the CTA was launched with: fewer than this would leave one of them waiting
    cudaFuncAttributes f;
    cudaError_t e = cudaFuncGetAttributes(&f, expanded_attend_kernel<DN, DV, BF>);
    if (e == cudaSuccess && f.numRegs * kAttendThreads < 256 * kSoftmaxRegs + 128 * kOtherRegs) e = cudaErrorInvalidConfiguration;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(expand_kernel<R, DN, DV, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ExpandSmem<R>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(expanded_attend_kernel<DN, DV, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ExpandedSmem<DN, DV>));
    return e;
}

template <int R, bool BF>
cudaError_t launch(const ExpandedArgs& a, int sm_count, cudaStream_t stream, int* launches) {
    if (a.m.Dn == 128)
        return a.m.Dv == 128 ? expand_and_attend<R, 128, 128, BF>(a, sm_count, stream, launches) : expand_and_attend<R, 128, 64, BF>(a, sm_count, stream, launches);
    return a.m.Dv == 128 ? expand_and_attend<R, 64, 128, BF>(a, sm_count, stream, launches) : expand_and_attend<R, 64, 64, BF>(a, sm_count, stream, launches);
}

template <int R, bool BF>
cudaError_t prepare(const Step& m) {
    if (m.Dn == 128) return m.Dv == 128 ? prepare<R, 128, 128, BF>() : prepare<R, 128, 64, BF>();
    return m.Dv == 128 ? prepare<R, 64, 128, BF>() : prepare<R, 64, 64, BF>();
}

}  // namespace

cudaError_t launch_expanded_plan(const ExpandedArgs& a, cudaStream_t stream, int* launches) {
    ++*launches;
    return pa::launch_dependent(expanded_plan_kernel, 1, 256, 0, stream, a);
}

cudaError_t launch_expanded(const ExpandedArgs& a, int dtype, int sm_count, cudaStream_t stream, int* launches) {
    if (dtype == PA_DTYPE_BF16) return a.m.R == 512 ? launch<512, true>(a, sm_count, stream, launches) : launch<256, true>(a, sm_count, stream, launches);
    return a.m.R == 512 ? launch<512, false>(a, sm_count, stream, launches) : launch<256, false>(a, sm_count, stream, launches);
}

cudaError_t prepare_expanded(const Step& m, int dtype) {
    if (dtype == PA_DTYPE_BF16) return m.R == 512 ? prepare<512, true>(m) : prepare<256, true>(m);
    return m.R == 512 ? prepare<512, false>(m) : prepare<256, false>(m);
}

}  // namespace latent
