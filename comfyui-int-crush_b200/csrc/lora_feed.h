// The producer of the streamed adapter kernels (lora_stream.cu): two rings of
// shared-memory stages, one block of the activations' side and then the
// adapters' blocks that meet it, one for each pass.  Plain C++, so that a host
// program can run it against every wait giving up.
#pragma once

#ifdef __CUDACC__
#define IC_FEED __device__ __forceinline__
#else
#define IC_FEED inline
#endif

namespace ic {

// The copies of a ring that may be in flight after `issued` of them: the last
// `stages`.  Where a copy's stage was taken again, its readers had released it.
template <class Landed>
IC_FEED void ring_drain(int issued, int stages, const Landed& landed) {
  for (int q = issued > stages ? issued - stages : 0; q < issued; ++q) landed(q);
}

// free_*(q): waits for the stage of copy q, false when it gave up; load_*:
// issues copy q; landed_*(q): waits for copy q.  Whether the feed ends by itself
// or gives up, every copy has landed when it returns: nothing may still write
// to the shared memory of a CTA that leaves, also when a reader gave up.
template <int SA, int SB, class FreeA, class LoadA, class LandedA, class FreeB, class LoadB, class LandedB>
IC_FEED void lora_feed(int blocks, int passes, const FreeA& free_a, const LoadA& load_a, const LandedA& landed_a,
                       const FreeB& free_b, const LoadB& load_b, const LandedB& landed_b) {
  int a = 0, b = 0;   // copies issued
  for (bool ok = true; ok && a < blocks;) {
    ok = free_a(a);
    if (!ok) break;
    load_a(a);
    ++a;
    for (int p = 0; p < passes; ++p) {
      ok = free_b(b);
      if (!ok) break;
      load_b(b, a - 1, p);
      ++b;
    }
  }
  ring_drain(a, SA, landed_a);
  ring_drain(b, SB, landed_b);
}

}  // namespace ic
