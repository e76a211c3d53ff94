// What a row of a masked step sees, on the CPU: lists of context tiles and words of bits against the rule, position by position.
#include <cstdio>
#include <random>
#include <vector>

#include "masked.cuh"

namespace {

bool in_window(int j, int row_pos, int W, int S) { return W == 0 || j < S || (long long)j > (long long)row_pos - W; }

template <int T>
bool lists(int ctx, int lo, int S) {
    const pa::VisTiles v = pa::vis_tiles<T>(ctx, lo, S);
    std::vector<char> listed((ctx + T - 1) / T, 0);
    int last = -1;
    for (int i = 0; i < v.count; ++i) {
        const int t = v.tile(i);
        if (t <= last || t >= (int)listed.size()) return false;
        last = t;
        listed[t] = 1;
    }
    // a tile is listed exactly when it holds a position that the row sees
    for (int t = 0; t < (int)listed.size(); ++t) {
        bool any = false;
        for (int j = t * T; j < ctx && j < (t + 1) * T; ++j) any |= j < S || j >= lo;
        if (any != (listed[t] != 0)) return false;
    }
    return true;
}

}  // namespace

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
    for (int round = 0; round < 200000; ++round) {
        const int past = pick(3) ? pick(700) : 0, n = 1 + pick(pick(2) ? 8 : 256), W = pick(4) ? 1 + pick(pick(2) ? 40 : 800) : 0, S = pick(3) ? pick(200) : 0;
        pa::MaskParams m{};
        m.window = W;
        m.sinks = S;
        const int tok = pick(n), ctx = past + tok + 1, lo = pa::window_lo(m, ctx), pos0 = 16 * pick(ctx / 16 + 3);
        const uint64_t w = pa::causal_bits(pos0, ctx, lo, S);
        for (int c = 0; c < 64; ++c) {
            const int j = pos0 + c;
            if (((w >> c) & 1) != (uint64_t)(j < ctx && in_window(j, ctx - 1, W, S))) { std::printf("word: past %d tok %d W %d S %d pos %d\n", past, tok, W, S, j); return 1; }
        }
        if ((uint32_t)w != pa::causal_bits32(pos0, ctx, lo, S)) { std::printf("the short word differs\n"); return 1; }
        if (!lists<32>(ctx, lo, S) || !lists<64>(ctx, lo, S)) { std::printf("tiles: ctx %d lo %d S %d\n", ctx, lo, S); return 1; }
        // a tree's bits at any offset
        uint32_t words[pa::kTreeWords];
        for (uint32_t& x : words) x = rng();
        const int o = pick(400) - 100;
        const uint64_t t = pa::tree_bits64(words, o);
        for (int c = 0; c < 64; ++c) {
            const int a = o + c;
            const uint64_t want = a >= 0 && a < pa::kTreeMax ? (words[a / 32] >> (a % 32)) & 1u : 0u;
            if (((t >> c) & 1) != want) { std::printf("tree bits at %d, bit %d\n", o, c); return 1; }
        }
        // a q tile's list covers what its rows see, and no half reaches beyond it
        const int G = 1 + pick(16), row0 = 256 * pick((n * G + 255) / 256);
        const bool tree = n <= pa::kTreeMax && pick(2);
        const pa::QTile q = pa::q_tile(m, past, n, G, row0, tree);
        for (int x = 0; x < 2; ++x) {
            const int r0 = row0 + 128 * x, r1 = std::min(row0 + 128 * x + 127, n * G - 1);
            if ((r0 >= n * G) != (q.cnt[x] == 0)) { std::printf("rows of half %d\n", x); return 1; }
            if (r0 >= n * G) continue;
            if (q.cnt[x] > q.v.count) { std::printf("half %d beyond the list\n", x); return 1; }
            for (int r : {r0, (r0 + r1) / 2, r1}) {
                const int p = tree ? past + pick(r / G + 1) : past + r / G, hi = tree ? past + n : p + 1;   // a token's depth is at most its index
                for (int j = 0; j < hi; ++j) {
                    if (!(j >= past && tree) && !in_window(j, p, W, S)) continue;
                    bool found = false;
                    for (int i = 0; i < q.cnt[x] && !found; ++i) found = q.v.tile(i) == j / 64;
                    if (!found) { std::printf("q tile: past %d n %d G %d row %d W %d S %d misses %d\n", past, n, G, r, W, S, j); return 1; }
                }
            }
        }
    }
    std::printf("ok\n");
    return 0;
}
