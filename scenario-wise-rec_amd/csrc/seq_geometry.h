// Launch geometry of the sequence-attention kernels (host only: no device code, compiles anywhere).
#pragma once
#include <cstdint>

// A launch: `blocks` workgroups (0: they do not fit a grid) for units x per_unit pieces of work, per_unit = tiles x inner; `rest` units behind
// the last write the rows of no sequence, at least 256 workgroups of their own; the units of an XCD go in rounds of `together` (sa_unit).
// A unit walks its column tiles in rounds of `tiles`, so any number of them is right: it is cut down where the grid would be too large.
// Computed once for a launch: workspaces and partial sums are laid out by `tiles`.
struct SaGrid {
    int tiles, per_unit, rest, together;
    unsigned blocks;
};
// workgroups of `threads` that a launch takes: a grid has fewer than 2^32 threads
static inline int64_t sa_most_blocks(int threads) { return ((1ll << 32) - 1) / threads; }
// tiles: column tiles of the longest sequence; inner: workgroups of a tile (heads x key ranges); together <= 0: all units in one round;
// threads: of a workgroup
static inline SaGrid sa_grid(int64_t units, int64_t tiles, int64_t inner, int64_t together, int threads) {
    SaGrid g{};
    int64_t per_unit = tiles * inner;
    const int64_t rest = (256 + per_unit - 1) / per_unit;
    const int64_t each = (units + rest + 7) / 8;                   // units of an XCD
    if (together <= 0 || together > each) together = each;
    const int64_t slots = (each + together - 1) / together * together;
    const int64_t room = sa_most_blocks(threads) / 8 / slots;                         // workgroups a unit may have
    if (inner > room) return g;
    if (per_unit > room) { tiles = room / inner; per_unit = tiles * inner; }
    g.tiles = static_cast<int>(tiles);
    g.per_unit = static_cast<int>(per_unit);
    g.rest = static_cast<int>(rest);
    g.together = static_cast<int>(together);
    g.blocks = static_cast<unsigned>(slots * 8 * per_unit);
    return g;
}
