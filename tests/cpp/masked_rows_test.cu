// What the row-by-row path of a masked step goes through, on the CPU: a row's tiles and its words of bits in them against the rule, position by position, for
// chunks and for trees of every shape (an ancestor is visible by its position in the tree, and lies where its token lies in the chunk).
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "masked.cuh"

namespace {

bool in_window(int j, int row_pos, int W, int S) { return W == 0 || j < S || (long long)j > (long long)row_pos - W; }

// Parents of n tokens: `kind` 0: anything in front; 1: near the token, a chain almost; 2: many children of one of the first tokens, then a chain; 3: a chain.
std::vector<int> tree(std::mt19937& rng, int n, int kind) {
    auto pick = [&](int k) { return (int)(rng() % (unsigned)k); };
    std::vector<int> p(n, -1);
    const int bush = 1 + pick(n), root = pick(4);
    for (int i = 1; i < n; ++i) {
        if (kind == 0) p[i] = pick(i + 1) - 1;
        else if (kind == 1) p[i] = std::max(0, i - 1 - pick(3));
        else if (kind == 2) p[i] = i <= root ? i - 1 : i < bush ? root : i - 1;
        else p[i] = i - 1;
    }
    return p;
}

}  // namespace

int main() {
    std::mt19937 rng(9);
    auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
    long long apart = 0;   // rows that see a token of the chunk in front of the place where their own window begins
    for (int round = 0; round < 3000; ++round) {
        const int past = pick(3) ? pick(pick(2) ? 12 : 300) : 0, n = 2 + pick(255), W = pick(5) ? 1 + pick(pick(2) ? 20 : 300) : 0, S = pick(4) ? pick(pick(2) ? 8 : 200) : 0;
        const bool is_tree = pick(4) != 0;
        pa::MaskParams m{};
        m.window = W;
        m.sinks = S;
        const std::vector<int> parent = tree(rng, n, pick(4));
        std::vector<int> depth(n);
        for (int i = 0; i < n; ++i) depth[i] = is_tree ? (parent[i] < 0 ? 0 : depth[parent[i]] + 1) : i;
        for (int i = 0; i < n; i += 1 + pick(5)) {
            const int at = past + depth[i];
            std::vector<char> sees(past + n, 0);
            uint32_t words[pa::kTreeWords] = {};
            for (int j = 0; j < past; ++j) sees[j] = in_window(j, at, W, S);
            for (int j = i; j >= 0; j = is_tree ? parent[j] : j - 1) {
                if (!in_window(past + depth[j], at, W, S)) continue;
                sees[past + j] = 1;
                words[j >> 5] |= 1u << (j & 31);
            }
            const pa::RowMask r = is_tree ? pa::RowMask{past, pa::window_lo(m, at + 1), words, past} : pa::RowMask{at + 1, pa::window_lo(m, at + 1), nullptr, past};
            const pa::VisTiles v = pa::row_tiles<32>(m, r, n);
            for (int j = past; is_tree && j < std::min(r.lo, past + n); ++j) apart += sees[j] && j / 32 >= (S + 31) / 32;
            int last = -1;
            for (int k = 0; k < v.count; ++k) {
                const int t = v.tile(k);
                if (t <= last) { std::printf("tiles out of order: past %d n %d row %d W %d S %d\n", past, n, i, W, S); return 1; }
                last = t;
                for (uint32_t w = pa::row_bits32(m, r, n, 32 * t); w; w &= w - 1) {
                    const int j = 32 * t + __builtin_ctz(w);
                    if (j >= past + n || !sees[j]) { std::printf("%s: past %d n %d row %d W %d S %d takes in %d\n", is_tree ? "tree" : "chunk", past, n, i, W, S, j); return 1; }
                    sees[j] = 0;
                }
            }
            for (int j = 0; j < past + n; ++j)
                if (sees[j]) { std::printf("%s: past %d n %d row %d W %d S %d misses %d\n", is_tree ? "tree" : "chunk", past, n, i, W, S, j); return 1; }
        }
    }
    // words of another sequence's: no position behind the row's own chunk
    for (int round = 0; round < 20000; ++round) {
        const int past = pick(200), n = 2 + pick(60);
        pa::MaskParams m{};
        m.window = pick(2) ? 1 + pick(50) : 0;
        m.sinks = pick(300);
        uint32_t words[pa::kTreeWords];
        for (uint32_t& w : words) w = rng();
        const pa::RowMask r{past, pa::window_lo(m, past + pick(256) + 1), words, past};
        const pa::VisTiles v = pa::row_tiles<32>(m, r, n);
        for (int k = 0; k < v.count; ++k)
            for (uint32_t w = pa::row_bits32(m, r, n, 32 * v.tile(k)); w; w &= w - 1)
                if (32 * v.tile(k) + __builtin_ctz(w) >= past + n) { std::printf("past %d n %d: a position behind the chunk\n", past, n); return 1; }
    }
    if (apart == 0) { std::printf("no row was drawn that sees a sink among its chunk\n"); return 1; }
    std::printf("ok\n");
    return 0;
}
