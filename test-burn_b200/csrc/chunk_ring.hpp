// The ring of K/V tiles of the ragged attention (chunk_attention.cu): which load goes where, who uses it, and how a stream
// walks it.  Plain C++, so that the host can run the walk against loads that land in any order.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MF_RING_FN __host__ __device__ __forceinline__
#else
#define MF_RING_FN inline
#endif

namespace mf {

// An item of n key tiles is 2 n loads, in the order in which the products want them:
//   paired rows   K0 V0 K1 V1 K2 V2 ...         both streams use every load
//   paired keys   K0 K1 V0 V1 K2 K3 V2 V3 ...   stream s uses tiles s, s + 2, ...; a last single tile is K V, stream 0's
// The loads of all items follow one another through the slots: load L is use L / slots of slot L % slots.
MF_RING_FN bool ring_uses(bool paired_rows, uint32_t n, uint32_t stream, uint32_t load)
{
    if (paired_rows) return true;
    return (load / 4) * 2 + 1 < n ? (load & 1u) == stream : stream == 0;
}
// The tile (from the item's first) whose V the load is; n or more: a K load.
MF_RING_FN uint32_t ring_v_tile(bool paired_rows, uint32_t n, uint32_t load)
{
    if (paired_rows) return load & 1u ? load / 2 : n;
    const uint32_t t = (load / 4) * 2;
    if (t + 1 < n) return load & 2u ? t + (load & 1u) : n;
    return load & 1u ? t : n;
}

// A stream's way through the ring.  It waits for EVERY load in turn, also for those that the other stream uses: a slot's
// barrier is waited for by parity, and a reader that leaves out a use cannot tell the use after it from the one before
// (with an odd number of slots the uses of a slot alternate between the streams).  A load that only the other stream uses
// is handed back as soon as it has landed, so that a slot is free after one arrival of each stream, whatever the form (and
// one of the warp that prepares V tiles, which goes through all loads, too).
template <uint32_t kSlots>
struct RingReader {
    uint32_t slot = 0, phase = 0;  // of the next load
    uint32_t load = 0;             // its number in the item
    // wait(slot, phase): until the load is there; pass(slot): this stream's arrival for a load it does not use.
    // Returns the slot of the stream's next load, which has landed.
    template <class Wait, class Pass>
    MF_RING_FN uint32_t next(bool paired_rows, uint32_t n, uint32_t stream, const Wait &wait, const Pass &pass)
    {
        for (;;) {
            const bool mine = ring_uses(paired_rows, n, stream, load);
            const uint32_t at = slot;
            wait(at, phase);
            if (!mine) pass(at);
            step();
            if (mine) return at;
        }
    }
    // Past the loads behind the stream's last one of the item.
    template <class Wait, class Pass>
    MF_RING_FN void finish(uint32_t n, const Wait &wait, const Pass &pass)
    {
        while (load < 2 * n) {
            wait(slot, phase);
            pass(slot);
            step();
        }
        load = 0;
    }
    // The phase of the load that next() has returned.
    MF_RING_FN uint32_t last_phase() const { return slot == 0 ? phase ^ 1 : phase; }
    MF_RING_FN void step()
    {
        ++load;
        if (++slot == kSlots) slot = 0, phase ^= 1;
    }
};

}  // namespace mf
