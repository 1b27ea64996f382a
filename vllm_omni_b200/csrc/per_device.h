// A positive number that is asked for once per device and kept, for one user of it (a kernel).  What could not be had (0 or less) is asked for again next time and
// stands in as `instead` meanwhile.
#pragma once

namespace omni {

struct PerDevice {
  int known[64] = {};
  template <typename Ask>
  int get(int device, int instead, Ask ask) {
    if (device < 0 || device >= 64) {
      const int n = ask();
      return n > 0 ? n : instead;
    }
    if (known[device] <= 0) known[device] = ask();
    return known[device] > 0 ? known[device] : instead;
  }
};

}  // namespace omni
