// A device handle with no device behind it, for the CPU tests of the argument checks: an entry point that refuses its
// arguments does so before it makes a HIP call, one that accepts them fails at its first HIP call where there is no GPU.
#include "../clpeak_amd/csrc/internal.h"

extern "C" mi355_dev *ffn_test_handle() {
  mi355_dev *d = new mi355_dev();
  d->ordinal = 0;
  d->props.num_cus = 256;
  return d;
}
