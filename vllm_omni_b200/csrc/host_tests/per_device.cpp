// PerDevice (per_device.h): what is asked for once, per user and per device, and what is asked for again (tests/test_lowbit_calls.py builds and runs this).
#include "../per_device.h"

int main() {
  omni::PerDevice a, b;
  int asked = 0;
  auto gives = [&](int n) { return [&asked, n] { ++asked; return n; }; };
  if (a.get(0, 74, gives(70)) != 70 || a.get(0, 74, gives(60)) != 70 || asked != 1) return 1;        // kept
  if (a.get(1, 74, gives(60)) != 60 || asked != 2) return 2;                                         // a device of its own
  if (b.get(0, 74, gives(50)) != 50 || asked != 3 || a.get(0, 74, gives(1)) != 70) return 3;         // a kernel of its own
  if (b.get(2, 74, gives(0)) != 74 || b.get(2, 74, gives(40)) != 40 || asked != 5) return 4;         // not to be had, then had
  if (b.get(64, 74, gives(9)) != 9 || b.get(-1, 74, gives(0)) != 74) return 5;                       // beyond what is kept
  return 0;
}
