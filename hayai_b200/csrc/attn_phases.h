// attn_phases.h -- rules of the many-row attention kernel's barriers, in plain C++: the kernel uses them, and
// a replay of the barriers' phases on the host (tests/attn_phases.cpp) checks them.
#pragma once

namespace hc {

// Key and value tiles of the ring.
constexpr int many_ring(bool i8, int head_dim) { return i8 ? 3 : head_dim == 64 ? 6 : 5; }

// May the rows' threads of a half wait for unit st's V tile before they have waited for its scores?  A wait by
// parity is sound only while the barrier is at the phase waited for or one before its end.  In a segment's
// later units this half has had the scores of the unit before, so the products' warp has waited for all tiles
// up to that unit's keys, and the tile that was in V's place before is one of them.  In a segment's first
// unit nothing says so: a half skips the segments that have no rows for it, and may be several of them, and
// any number of phases, ahead of the copies.  There it waits for the scores first: they are issued after all
// tiles up to this unit's keys were waited for.
constexpr bool many_early_look(int st, int lo) { return st > lo; }

}  // namespace hc
