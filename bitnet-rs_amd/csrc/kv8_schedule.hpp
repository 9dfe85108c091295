// kv8_schedule.hpp -- when k_kv8_prefill's walk over tiles of keys reads and writes its two buffers of LDS (host code only).
//
// An iteration works on tile i in two halves of 32 keys and begins with its only barrier, so that the waves of a group may be a whole iteration apart: what one of them writes must not be read or
// written by another one between the same two barriers.  Tile j lies in buffer j % 2; its keys' scales in slot j / 2 % 2 of it besides.
//
//   iteration i   reads                                                              writes
//   half 0        keys 32 .. 63 of tile i and their scales, values, factors          factors (their exponents among them) and values of tile i + 1
//   half 1        keys 0 .. 31 of tile i + 1 and their scales, values, factors       keys 0 .. 31 of tile i + 2 and the scales of all its keys, keys 32 .. 63 of tile i + 1
//                 of tile i
//
// Keys 32 .. 63 of tile i + 2 would go where those of tile i are read.  The kernel takes what it writes from kKv8Schedule, and kv8_schedule_holds goes through the table for it.
#pragma once

namespace bitnet_hip {

struct Kv8Schedule {  // how many tiles ahead of the iteration's own that tile is whose .. are written
    int keys[2];      // keys 0 .. 31 and 32 .. 63
    int scales, values, factors;
    int slots;  // of a buffer's scales
};
constexpr Kv8Schedule kKv8Schedule = {{2, 1}, 2, 1, 1, 2};

enum Kv8Region { kKv8Keys0, kKv8Keys1, kKv8Scales, kKv8Values, kKv8Factors, kKv8Regions };
struct Kv8Access {
    int region, tile;
    bool writes;
};
constexpr int kKv8Accesses = 11;

constexpr int kv8_place(const Kv8Schedule &s, const Kv8Access &a) { return a.tile % 2 + (a.region == kKv8Scales && s.slots == 2 ? a.tile / 2 % 2 * 2 : 0); }
// Nothing is written between the barriers where its place is read or written otherwise, and what is read was written last ahead of the barrier.
constexpr bool kv8_schedule_holds(const Kv8Schedule &s) {
    int holds[kKv8Regions][4] = {};  // the tile in a place, behind the barrier of iteration i
    for (int i = 0; i < 16; ++i) {
        const Kv8Access now[kKv8Accesses] = {{kKv8Keys1, i, false}, {kKv8Keys0, i + 1, false}, {kKv8Scales, i, false}, {kKv8Scales, i + 1, false}, {kKv8Values, i, false}, {kKv8Factors, i, false},
                                             {kKv8Keys0, i + s.keys[0], true}, {kKv8Keys1, i + s.keys[1], true}, {kKv8Scales, i + s.scales, true}, {kKv8Values, i + s.values, true},
                                             {kKv8Factors, i + s.factors, true}};
        for (int a = 0; a < kKv8Accesses; ++a) {
            for (int b = 0; b < kKv8Accesses; ++b)
                if (a != b && now[b].writes && now[b].region == now[a].region && kv8_place(s, now[b]) == kv8_place(s, now[a])) return false;
            if (!now[a].writes && i >= 4 && holds[now[a].region][kv8_place(s, now[a])] != now[a].tile) return false;  // (every place has been written from here on)
        }
        for (const Kv8Access &a : now)
            if (a.writes) holds[a.region][kv8_place(s, a)] = a.tile;
    }
    return true;
}
static_assert(kv8_schedule_holds(kKv8Schedule), "k_kv8_prefill: a place in LDS is written between the barriers where it is read");

}  // namespace bitnet_hip
