// Copies into a ring of N places, each place with a barrier whose phase ends when its copy has landed: what a warp that gives up has to wait for
// before its block's memory may become another's.  Plain C++: the waits come from the caller, ``wait(place, parity)`` (whether the phase of that
// parity has ended, after a limited time).
#pragma once
#ifdef __CUDACC__
#define I4_BOTH __host__ __device__ __forceinline__
#else
#define I4_BOTH inline
#endif

// A ring in which tiles may be passed over (nothing is copied for them): tile i's place is i % N, and the place's phase is counted.
template <int N> struct I4Ring {
    unsigned phase = 0;                  // parity of the phase that a place is in, a bit a place
    // Waits for a tile's copy.  Only one that landed ends its place's phase.
    template <typename Wait> I4_BOTH bool landed(int tile, Wait wait) {
        if (!wait(tile % N, (phase >> (tile % N)) & 1u)) return false;
        phase ^= 1u << (tile % N);
        return true;
    }
    // Waits for what is under way when the tiles before ``tile`` have been dealt with: of it and the N - 1 behind it, those that were asked for.
    template <typename Asked, typename Wait> I4_BOTH void drain(int tile, Asked asked, Wait wait) const {
        for (int i = tile; i < tile + N; ++i)
            if (asked(i)) wait(i % N, (phase >> (i % N)) & 1u);
    }
};

// A ring that every tile takes in turn, tile i's phase being the (i / N)-th of its place: waits for the last copies of the ``issued`` ones, those that
// may be under way when nobody is known to have waited for them (which returns at once for all that landed).
template <int N, typename Wait> I4_BOTH void i4_drain(int issued, Wait wait) {
    for (int i = issued > N ? issued - N : 0; i < issued; ++i) wait(i % N, (unsigned)(i / N) & 1u);
}
