// The order of a row's classes, on the host: Places::upto keeps the classes whose places reach a border, for
// borders at, between and next to the keys that logits have.
#include "kernels/row_select.h"

#include <cstdio>
#include <limits>
#include <vector>

using namespace mlapi::lrow;

int main() {
  typedef std::numeric_limits<float> lim;
  const float logits[] = {-lim::infinity(), -lim::max(), -2.f, -1.f, -lim::min(), -lim::denorm_min(), -0.f, 0.f,
                          lim::denorm_min(), lim::min(), 1.f, 1.5f, lim::max(), lim::infinity()};
  std::vector<uint32_t> keys = {KEY_MASKED + 1, KEY_BELOW_ZERO - 1, KEY_BELOW_ZERO, KEY_BELOW_ZERO + 1};
  const uint32_t most = order_key(lim::infinity());
  for (float z : logits)
    for (int d = -1; d <= 1; ++d) {
      const uint32_t k = order_key(z) + (uint32_t)d;
      if (k > KEY_MASKED && k <= most) keys.push_back(k);
    }
  long wrong = 0, tried = 0;
  for (int K : {1, 2, 5, 64, 4096, 1 << 20}) {
    const Places places(K);
    const int picks[] = {0, 1, 2, K / 3, K / 2, K - 2, K - 1};
    for (uint32_t key : keys)
      for (int low : picks) {
        if (low < 0 || low >= K) continue;
        const uint64_t border = places.of(key, low);
        float z;
        int last;
        places.upto(border, z, last);
        for (float x : logits)
          for (int i : picks) {
            if (i < 0 || i >= K || order_key(x) <= KEY_MASKED) continue;
            const bool in = x > z || (x == z && i <= last), want = places.of(order_key(x), i) >= border;
            ++tried;
            if (in != want && ++wrong <= 5)
              printf("K %d border key %08x class %d: logit %g class %d kept %d, not %d\n", K, key, low, x, i, in, want);
          }
      }
  }
  printf("%ld of %ld wrong\n", wrong, tried);
  return wrong != 0 || tried == 0;
}
