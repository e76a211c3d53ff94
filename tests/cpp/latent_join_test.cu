// The records by which the join of latent attention's absorbed form finds a row's partial results, on the CPU: what the attention writes comes
// through as it is, and whatever else may lie in the scratch leads nowhere outside it.
#include <climits>
#include <cstdio>
#include <random>

#include "latent_kernels.h"

static int fail(const char* what, int2 part, int step, long long rows) {
    std::printf("%s: first %d, pieces %d, step %d, rows %lld\n", what, part.x, part.y, step, rows);
    return 1;
}

int main() {
    std::mt19937_64 rng(7);
    const int edges[] = {INT_MIN, INT_MIN + 1, -65, -1, 0, 1, 2, 63, 64, 74, 148, 149, 9471, 9472, 9473, INT_MAX - 128, INT_MAX - 1, INT_MAX};
    const int steps[] = {latent::kTile, 2 * latent::kTile};
    for (int step : steps)
        for (long long slots : {1LL, 2LL, 75LL, 148LL, 4096LL, 33554431LL}) {
            const long long rows = slots * latent::kTile;
            const auto garbage = [&](int x, int y) {
                const int2 part = latent::checked_part(make_int2(x, y), step, rows);
                // every index that the join takes from the record
                if (part.y < 0) return fail("negative", part, step, rows);
                if (part.y > 0 && (part.x < 0 || part.x >= rows || part.x + (part.y - 1LL) * step >= rows)) return fail("outside", part, step, rows);
                return 0;
            };
            for (int x : edges)
                for (int y : edges)
                    if (garbage(x, y)) return 1;
            for (int k = 0; k < 200000; ++k)
                if (garbage((int)rng(), (int)(rng() >> (rng() & 31)))) return 1;
            // what the attention writes: row e of a slot, one result in each of the groups from there on
            const int row_tiles = step / latent::kTile;
            for (int k = 0; k < 20000; ++k) {
                const long long slot = rng() % slots, most = (slots - 1 - slot) / row_tiles + 1;
                const int2 part = make_int2((int)(slot * latent::kTile + rng() % latent::kTile), (int)(1 + rng() % most));
                const int2 same = latent::checked_part(part, step, rows);
                if (same.x != part.x || same.y != part.y) return fail("a good record is refused", part, step, rows);
            }
        }
    std::puts("ok");
    return 0;
}
