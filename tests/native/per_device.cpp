// PerDevice against a fake of the calls that it stands in front of.
#include <stdio.h>

#include "hipress/per_device.h"

static int current = 0, calls[70] = {}, fail = 0;
static hipress::PerDevice state;

static int use(int device, int* value) {
  current = device;
  return state.get(device, [](int* v) {
    ++calls[current];
    if (fail) return 1;
    *v = 100 + current;
    return 0;
  }, value);
}

#define CHECK(x) if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; }

int main() {
  int v = 0;
  fail = 1;
  CHECK(use(0, &v) == 1 && calls[0] == 1);          // a failure is told, and not remembered
  fail = 0;
  CHECK(use(0, &v) == 0 && v == 100 && calls[0] == 2);
  CHECK(use(1, &v) == 0 && v == 101 && calls[1] == 1);   // the second device is asked for itself
  fail = 1;
  CHECK(use(0, &v) == 0 && v == 100 && calls[0] == 2);   // both are known
  CHECK(use(1, &v) == 0 && v == 101 && calls[1] == 1);
  CHECK(use(2, &v) == 1 && use(0, &v) == 0);
  fail = 0;
  CHECK(use(63, &v) == 0 && v == 163 && use(63, &v) == 0 && calls[63] == 1);
  CHECK(use(64, &v) == 0 && v == 164 && use(64, &v) == 0 && v == 164 && calls[64] == 2);   // beyond what is remembered
  printf("per device ok\n");
  return 0;
}
