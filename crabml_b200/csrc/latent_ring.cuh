// latent_ring.cuh -- what the kernels of the latent attention wait for, in so far as it is tested without a GPU.  No CUDA call in here.
//
// The ring of cached rows of latent_rows_kernel (latent_attn.cu): which slot a step's rows lie in and which barrier says that they have come.
// LR_GROUPS groups of warps take a run's steps by turns; step j lies in slot j % slots.  A wait by parity tells a phase from its neighbours only, so it needs a waiter that has seen the phase
// before.  With a barrier a slot and an odd number of slots, step j + slots is another group's than step j: where the copy of j came late, that group's wait succeeded on the phase before j's and
// it read the slot's old rows.  So a step has one of LR_GROUPS * slots barriers: the one before it there is step j - LR_GROUPS * slots, which the same group has waited for.
#pragma once

#ifdef __CUDACC__
#define LR_FN __host__ __device__ __forceinline__
#else
#define LR_FN inline
#endif
#define LR_GROUPS 2
#define LR_SLOTS 8                            // most slots of the ring,
#define LR_SLOTS_LEAST 3                      // .. and least: a group asks for step j + slots when it has step j + LR_GROUPS

struct LrPlace { int slot, bar; unsigned parity; };
LR_FN LrPlace lr_place(int step, int slots) {
    const int turn = step / (LR_GROUPS * slots), bar = step - turn * LR_GROUPS * slots;
    return {bar < slots ? bar : bar - slots, bar, (unsigned)turn & 1u};
}
static_assert(LR_GROUPS == 2, "a barrier's place in the ring");

// Rounds of several warps that meet at barriers within a round.  A warp whose wait ran out, or that saw that another one's had, stays for the rounds that are left (without its loads and stores):
// warps see it at different times, and one that left its loop would be waited for at the others' barriers for good
template <class Wait, class Body>
LR_FN void lt_rounds(int lo, int hi, Wait wait, Body body) {
    bool ok = true;
    for (int i = lo; i < hi; i++) {
        ok = ok && wait(i);
        body(i, ok);
    }
}
