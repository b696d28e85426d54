// Blocks of one launch that hand data to whichever of them arrives last (gfx950 only).
#pragma once

#include <atomic>

#include "common.h"

namespace mesh_moe {

// Accesses that are coherent across the GPU's compute dies without a cache
// flush.  Each die (XCD) has its own L2; an ordinary store may sit there, and
// an ordinary load may hit a stale line there, until a device-scope fence
// writes back / invalidates that whole L2 -- too expensive to issue from
// every block of a kernel whose other blocks are still streaming through the
// same L2.  A relaxed atomic store / load at device scope is a write-through
// store / a load that bypasses lines the L2 cannot vouch for.  Blocks of one
// launch exchange their data only through these: the writer waits until its
// stores have completed (vmcnt 0) before it bumps the arrival counter, the
// reader loads after it has seen the counter.
template <typename T>
__device__ __forceinline__ void st_dev(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T ld_dev(const T* p) {
  return __hip_atomic_load(const_cast<T*>(p), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
// this wavefront's global stores (and loads) have completed
__device__ __forceinline__ void wait_stores() {
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0), nothing else
  asm volatile("" ::: "memory");
}

// A counter is a 64-bit word: call number << 16 | arrivals.  A word that does
// not carry the current call's number counts as zero, so the workspace may
// hold anything when the call starts; the last arrival leaves zero behind.

// Puts a counter word into this call's state "no arrivals yet", whatever it holds: zero
// where the last arrival of a call left it, anything where the workspace's memory has
// served something else since (between two passes of a training step it has).  One
// thread of a block that arrives at the word itself; it hands the returned word to
// counter_settle once its work is done (nobody waits for it before) and arrives behind
// that.
__device__ __forceinline__ unsigned long long counter_prepare(
    unsigned long long* word, unsigned long long call) {
  return __hip_atomic_exchange(word, call << 16, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
}

// Puts back the arrivals that came before counter_prepare.  Until then the word counts
// too few, so no arrival takes itself for the last one, and this block's own arrival is
// still to come.
__device__ __forceinline__ void counter_settle(unsigned long long* word,
                                               unsigned long long call,
                                               unsigned long long prepared) {
  if ((prepared >> 16) == call)
    (void)__hip_atomic_fetch_add(word, prepared & 0xffffu, __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT);
}

// true for the last of `expected` arrivals; one thread per arrival.  The
// common case is one fetch-add on a word that counter_prepare stamped long
// ago.  An arrival that finds another stamp (its add then changed a word
// nobody relies on) installs the stamp itself or, if somebody else just did,
// adds again: every arrival ends with exactly one successful operation on a
// word that carries this call's stamp.
__device__ __forceinline__ bool arrive_is_last(unsigned long long* word,
                                               unsigned long long call,
                                               unsigned expected) {
  unsigned long long old = __hip_atomic_fetch_add(
      word, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if ((old >> 16) == call) return (unsigned)((old + 1) & 0xffffu) == expected;
  old = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (;;) {
    if ((old >> 16) == call) {
      old = __hip_atomic_fetch_add(word, 1ull, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
      return (unsigned)((old + 1) & 0xffffu) == expected;
    }
    const unsigned long long seen = atomicCAS(word, old, (call << 16) | 1ull);
    if (seen == old) return expected == 1u;
    old = seen;
  }
}

// Number of a call whose blocks arrive at counters: what its workspace holds is read
// relative to it.
inline unsigned long long next_call_number() {
  static std::atomic<unsigned long long> counter{1};
  unsigned long long n = counter.fetch_add(1, std::memory_order_relaxed);
  return (n & ((1ull << 48) - 1)) | (1ull << 47);
}

}  // namespace mesh_moe
