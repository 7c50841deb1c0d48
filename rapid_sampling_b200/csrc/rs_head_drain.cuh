// What is still to be awaited when a product kernel stops early: which steps of a ring of stages, by plain arithmetic that the
// host can run too.
#pragma once
#include <stdint.h>
#ifdef __CUDACC__
#define RS_DRAIN_FN __host__ __device__ __forceinline__
#else
#define RS_DRAIN_FN inline
#endif

namespace rs {

struct DrainSteps {      // [from, to)
    uint32_t from, to;
};
// Step k uses slot k % ring, and its use is the slot's phase k / ring, of which a wait wants the parity.
RS_DRAIN_FN uint32_t drain_slot(uint32_t k, uint32_t ring) { return k % ring; }
RS_DRAIN_FN uint32_t drain_parity(uint32_t k, uint32_t ring) { return (k / ring) & 1u; }
// Of n steps in all, those whose slots nothing has used since.
RS_DRAIN_FN DrainSteps drain_recent(uint32_t n, uint32_t ring) { return {n > ring ? n - ring : 0u, n}; }
// A pair's copies of a step count on one barrier, which wants an arrival of either CTA: those that this CTA owes, so that the
// other's copies of these steps can be awaited.  The slots' uses before were complete: the other CTA, which went on to step k,
// had seen the products of step k - ring, and those had waited for both CTAs' copies.
RS_DRAIN_FN DrainSteps drain_owed(uint32_t mine, uint32_t other) { return {mine, other > mine ? other : mine}; }

}  // namespace rs
