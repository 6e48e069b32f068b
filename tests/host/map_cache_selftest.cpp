// The table of tensor maps (map_cache.hpp): what it keeps and what it forgets, and that threads with the same and with other keys
// never get one another's maps.
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>

#include "../../catccos_b200/csrc/map_cache.hpp"

using namespace catccos;

struct alignas(64) Map {
    uint64_t word[16];
};

static MapKey key_of(uint64_t i) { return {reinterpret_cast<const void*>(0x1000 + 64 * i), 128 + i, 7 * i, 64, 32, i % 3 == 0, 1, i % 5}; }

static int encode(uint64_t i, Map* m)
{
    for (uint64_t w = 0; w < 16; ++w) {
        m->word[w] = i * 1000 + w;
    }
    return 0;
}

static bool is(uint64_t i, const Map& m)
{
    for (uint64_t w = 0; w < 16; ++w) {
        if (m.word[w] != i * 1000 + w) {
            return false;
        }
    }
    return true;
}

#define EXPECT(x)                                 \
    if (!(x)) {                                   \
        printf("line %d: %s\n", __LINE__, #x);    \
        return 1;                                 \
    }

int main()
{
    MapCache<Map>& maps = thread_maps<Map>();
    int made = 0;
    Map m;
    auto get = [&](uint64_t i) { return maps.get(key_of(i), &m, [&](Map* out) { return ++made, encode(i, out); }); };
    for (int round = 0; round < 3; ++round) {
        for (uint64_t i = 0; i < (uint64_t)kMapCacheSize; ++i) {
            EXPECT(get(i) == 0 && is(i, m));
        }
    }
    EXPECT(made == kMapCacheSize);
    EXPECT(get(0) == 0 && get(100) == 0 && is(100, m) && made == kMapCacheSize + 1);  // takes the place of key 1, the oldest
    EXPECT(get(0) == 0 && is(0, m) && made == kMapCacheSize + 1);
    EXPECT(get(1) == 0 && is(1, m) && made == kMapCacheSize + 2);
    // a map that cannot be made is not kept
    EXPECT(maps.get(key_of(200), &m, [](Map*) { return -3; }) == -3);
    EXPECT(maps.get(key_of(200), &m, [](Map* out) { return encode(200, out); }) == 0 && is(200, m));

    std::atomic<int> wrong{0}, ready{0};
    std::vector<std::thread> threads;
    for (uint64_t t = 0; t < 8; ++t) {
        threads.emplace_back([&, t] {
            ready++;
            while (ready < 8) {
            }
            uint64_t at = t;
            for (int n = 0; n < 300000; ++n) {
                at = at * 6364136223846793005ull + 1442695040888963407ull;
                const uint64_t i = (at >> 33) % 24;
                Map got;
                thread_maps<Map>().get(key_of(i), &got, [&](Map* out) { return encode(i, out); });
                wrong += is(i, got) ? 0 : 1;
            }
        });
    }
    for (std::thread& t : threads) {
        t.join();
    }
    EXPECT(wrong == 0);
    printf("map cache ok\n");
    return 0;
}
