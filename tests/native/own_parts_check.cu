// own_parts (decode_stream.cuh) on the host: where the parts of a pair lie, for every place it may have, and for
// places that were never written.  Prints the names of the checks that hold.
#include <cstdint>
#include <cstdio>
#include <random>

#include "decode_stream.cuh"

using namespace mllm_b200;

static bool all_places() {   // the CTAs found are those whose tiles meet the pair's, and no others
    const int ctas = 7;
    for (int per = 1; per <= 4; ++per)
        for (int p0 = 0; p0 < ctas * per; ++p0)
            for (int tiles = 1; p0 + tiles <= ctas * per; ++tiles) {
                int first, count, want_first = -1, want = 0;
                for (int c = 0; c < ctas; ++c)
                    if (c * per < p0 + tiles && (c + 1) * per > p0) {
                        if (want++ == 0) want_first = c;
                    }
                if (!own_parts(p0, tiles, per, ctas, &first, &count) || first != want_first || count != want) return false;
            }
    return true;
}

static bool no_tiles() {
    int first, count;
    return own_parts(-5, 0, 3, 7, &first, &count) && first == 0 && count == 0;
}

static bool any_bytes() {   // whatever lies there, no slot outside the workspace is named
    std::mt19937 rng(1);
    for (int shared = 0; shared < 2; ++shared)
        for (int i = 0; i < 2000000; ++i) {
            const int ctas = 1 + (int)(rng() % 320), most = most_ctas(ctas, shared), per = 1 + (int)(rng() % 1000);
            const int tiles = 1 + (int)(rng() % 0x7ffeffff);
            const int p0 = i % 3 ? (int)rng() : (int)(rng() % (8 * ctas * per));
            int first, count;
            const bool ok = own_parts(p0, tiles, per, most, &first, &count);
            if (first < 0 || count < 0 || (int64_t)first + count > most || ok != (count >= 1)) return false;
        }
    int first, count;   // 4 * ctas slots only where the prefix's decode has them; a sum beyond 31 bits
    return !own_parts(300, 10, 1, most_ctas(296, 0), &first, &count) && own_parts(300, 10, 1, most_ctas(296, 1), &first, &count) &&
           !own_parts(0x7fffffff, 10, 1, most_ctas(296, 1), &first, &count);
}

int main() {
    bool ok = true;
    auto check = [&](const char* name, bool holds) {
        if (holds) printf("%s\n", name);
        ok = ok && holds;
    };
    check("all_places", all_places());
    check("no_tiles", no_tiles());
    check("any_bytes", any_bytes());
    return ok ? 0 : 1;
}
