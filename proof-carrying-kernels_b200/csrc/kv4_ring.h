// The order in which a warp of the 4-bit attention waits for, uses and issues the copies of its ring
// (no CUDA in it, so that a test can run it on the host).
#pragma once

#ifdef __CUDACC__
#define PCK_RING_FN __device__ __forceinline__
#else
#define PCK_RING_FN inline
#endif

namespace pck {

// Takes `stages` stages through `kSlots` slots; the copies of the first min(kSlots, stages) are on their way.
// wait(slot) is false if it gave up: then nothing more is used or issued, but what is on its way is still
// waited for, since a copy must not land in shared memory that has been given up. Returns false after that.
template <int kSlots, typename Wait, typename Use, typename Issue>
PCK_RING_FN bool take_stages(int stages, Wait wait, Use use, Issue issue) {
  auto after = [](int slot) { return slot + 1 == kSlots ? 0 : slot + 1; };
  int slot = 0;
  for (int k = 0; k < stages; ++k) {
    if (!wait(slot)) {
      for (int i = 1; i < kSlots && k + i < stages; ++i) wait(slot = after(slot));
      return false;
    }
    use(k, slot);
    if (k + kSlots < stages) issue(k + kSlots, slot);
    slot = after(slot);
  }
  return true;
}

}  // namespace pck
