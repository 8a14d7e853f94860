// How a kernel's warps share the registers that its block was launched with.
// Plain C++, so that a host program can check it.
#pragma once

namespace ic {

// `few_threads` keep `few` registers each (setmaxnreg.dec), `many_threads` go on with
// `many` (setmaxnreg.inc).  The increase waits, without a limit, until the block has
// that many to spare: a kernel that was compiled to fewer a thread than the split
// adds up to must not be launched.
struct RegisterSplit {
  int few_threads, few, many_threads, many;
  constexpr bool fits(int registers) const {   // a thread, as compiled; given out in eights
    return (registers + 7) / 8 * 8 * (few_threads + many_threads) >= few_threads * few + many_threads * many;
  }
};

}  // namespace ic
