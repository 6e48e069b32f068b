// The tensor maps of a thread's last operands.
//
// A tensor map depends on (address, extents, box) only; a decode loop calls with the same few buffers over and over, and an
// encode costs about as much as the launch it precedes.  A small most-recently-used table keeps the last maps.  Every host
// thread has a table of its own: calls of several threads run at the same time (the calls on torch tensors let go of the
// interpreter's lock), and a map that one thread reads while another replaces it would send a kernel to other memory.
#pragma once

#include <cstdint>

namespace catccos {

struct MapKey {
    const void* base;
    uint64_t inner, outer;
    uint32_t box_inner, box_outer;
    bool fp4;
    uint32_t elem;
    uint64_t pitch;
    uint32_t depth = 0;  // matrices of a map with three axes, 0: two axes
    uint64_t plane = 0;  // bytes from one of them to the next
    bool operator==(const MapKey& o) const
    {
        return base == o.base && inner == o.inner && outer == o.outer && box_inner == o.box_inner &&
               box_outer == o.box_outer && fp4 == o.fp4 && elem == o.elem && pitch == o.pitch && depth == o.depth && plane == o.plane;
    }
};

constexpr int kMapCacheSize = 16;

template <typename Map>
struct MapCache {
    MapKey key[kMapCacheSize] = {};
    Map map[kMapCacheSize] = {};
    uint64_t used[kMapCacheSize] = {};
    uint64_t clock = 0;

    // The key's map: the one that is kept, or the one that encode(map) makes.  A map that could not be made is not kept; the
    // code is encode's.
    template <typename Encode>
    int get(const MapKey& k, Map* out, Encode&& encode)
    {
        int victim = 0;
        for (int i = 0; i < kMapCacheSize; ++i) {
            if (used[i] != 0 && key[i] == k) {
                used[i] = ++clock;
                *out = map[i];
                return 0;
            }
            if (used[i] < used[victim]) {
                victim = i;
            }
        }
        const int rc = encode(out);
        if (rc == 0) {
            key[victim] = k;
            map[victim] = *out;
            used[victim] = ++clock;
        }
        return rc;
    }
};

template <typename Map>
MapCache<Map>& thread_maps()
{
    static thread_local MapCache<Map> maps;
    return maps;
}

}  // namespace catccos
