// What pa_b200_latent_reserve makes room for, on the CPU (host code only, no device is touched): the scratch of every step of no more tokens,
// sequences and block indices in the same form, and after an AUTO reserve in either of the two forms.
#include <cstdio>
#include <random>

#include "latent_api.cu"

static int checked = 0;

static bool holds(const pa_latent_handle& h, int form, int T, int S, int B, int call, int t, int s, int b) {
    ++checked;
    const size_t room = reserved_bytes(&h, T, S, B, form), need = plan_scratch(&h, t, s, b, call).total;
    if (need <= room) return true;
    const pa_latent_desc& d = h.desc;
    std::printf("%d heads, %d/%d/%d/%d, blocks of %d: reserve(%d, %d, %d, form %d) holds %zu bytes, attend(%d, %d, %d, form %d) needs %zu\n", d.num_heads, d.latent_size,
                d.rope_size, d.nope_size, d.value_size, d.block_size, T, S, B, form, room, t, s, b, call, need);
    return false;
}

int main() {
    std::mt19937_64 rng(11);
    const auto below = [&](long long n) { return (long long)(rng() % (unsigned long long)n); };
    const auto spread = [&](int bits) { return (int)(rng() >> (64 - 1 - below(bits))); };      // over the logarithm
    pa_latent_handle h;
    h.desc = pa_latent_desc{sizeof(pa_latent_desc), 128, 512, 64, 128, 128, 64, PA_DTYPE_BF16};
    // by hand: a narrower form, and fewer blocks that let more heads into a pass
    bool ok = holds(h, PA_LATENT_AUTO, 4096, 2, 64, PA_LATENT_ABSORBED, 4096, 2, 64) && holds(h, PA_LATENT_AUTO, 4096, 1, 64, PA_LATENT_ABSORBED, 4096, 1, 64) &&
              holds(h, PA_LATENT_EXPANDED, 2048, 64, 20000, PA_LATENT_EXPANDED, 2048, 64, 16000) && holds(h, PA_LATENT_EXPANDED, 2048, 64, 16384, PA_LATENT_EXPANDED, 2048, 64, 12000);
    for (int k = 0; ok && k < 300000; ++k) {
        static const int kHeads[] = {1, 2, 3, 8, 16, 40, 64, 100, 128, 147, 148, 149, 200, 296, 297, 1024};
        h.sm_count = k % 7 == 0 ? 132 : 148;
        h.desc.num_heads = kHeads[below(16)];
        h.desc.latent_size = 256 << below(2); h.desc.rope_size = 32 << below(2); h.desc.nope_size = 64 << below(2); h.desc.value_size = 64 << below(2);
        h.desc.block_size = 16 << below(3);
        const int T = spread(16), S = spread(12), B = spread(20);
        const int t = k % 3 ? (int)below(T + 1) : T, s = k % 5 ? (int)below(S + 1) : S, b = k % 2 ? (int)below(B + 1) : B;
        const int form = (int)below(3), call = form == PA_LATENT_AUTO ? (int)below(3) : form;
        ok = holds(h, form, T, S, B, call, t, s, b);
    }
    // the parts of a step's scratch lie beside one another, inside it
    for (int k = 0; ok && k < 20000; ++k) {
        h.desc.num_heads = 1 + (int)below(300);
        const Scratch x = plan_scratch(&h, 1 + spread(14), 1 + spread(10), spread(18), PA_LATENT_EXPANDED);
        const size_t key = (size_t)x.heads * x.rows * h.desc.nope_size * 2, value = (size_t)x.heads * x.rows * h.desc.value_size * 2;
        ok = x.heads >= 1 && x.heads <= h.desc.num_heads && x.k % 1024 == 0 && x.v % 1024 == 0 && x.k + key <= x.v && x.v + value <= x.total && x.part_slots <= 2 * h.sm_count &&
             x.k_rope + (size_t)x.rows * 128 <= x.k;
        if (!ok) std::printf("parts of the scratch overlap\n");
    }
    if (ok) std::printf("ok: %d\n", checked);
    return ok ? 0 : 1;
}
