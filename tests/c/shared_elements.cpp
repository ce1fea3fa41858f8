// Which strided tensors share elements (csrc/attention/overlap.hpp): small ones against every pair of elements, and large
// ones that programs have.
#include <attention/overlap.hpp>

#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

using namespace certex_amd::attention;
using tensor = std::vector<dimension>;

std::vector<int64_t> offsets(tensor const& t)
{
  std::vector<int64_t> at{0};
  for (dimension d : t) {
    std::vector<int64_t> next;
    for (int64_t o : at) {
      for (int64_t i = 0; i < d.n; ++i) { next.push_back(o + i * d.stride); }
    }
    at = next;
  }
  return at;
}

void expect(bool ok, const char* what)
{
  if (!ok) {
    std::printf("%s\n", what);
    std::exit(1);
  }
}

bool two(tensor const& a, tensor const& b, int64_t distance)
{
  return shares(a.data(), int(a.size()), b.data(), int(b.size()), distance);
}

int main()
{
  std::mt19937 rng(1);
  const auto draw = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  int selves = 0, pairs = 0;
  for (int i = 0; i < 40000; ++i) {
    tensor a, b;
    for (int d = draw(1, 4); d > 0; --d) { a.push_back({draw(1, 4), draw(0, 14)}); }
    for (int d = draw(1, 4); d > 0; --d) { b.push_back({draw(1, 4), draw(0, 3) > 0 ? a[draw(0, int(a.size()) - 1)].stride : draw(0, 14)}); }
    const auto x = offsets(a), y = offsets(b);
    const std::set<int64_t> xs(x.begin(), x.end());
    const bool self = xs.size() < x.size();
    expect(shares_itself(a.data(), int(a.size())) == self, "a tensor and itself");
    const int64_t distance = draw(-30, 30);
    bool met               = false;
    for (int64_t o : y) { met = met || xs.count(o + distance) > 0; }
    expect(two(a, b, distance) == met, "two tensors");
    selves += self;
    pairs += met;
  }
  expect(selves > 4000 && selves < 36000 && pairs > 4000 && pairs < 36000, "cases of both answers");

  // slices of one projection, tokens of 6,144 elements: heads of 128 beside one another, and one element off
  const tensor q{{100000, 6144}, {32, 128}, {128, 1}}, k{{100000, 6144}, {8, 128}, {128, 1}};
  expect(!two(q, k, 4096) && !two(k, q, -4096) && two(q, k, 4095) && two(k, q, -4095), "slices of a projection");
  expect(!two(q, q, 6144 * 100000) && two(q, q, 6144) && two(q, q, 1) && two(q, q, 0), "a tensor and the next");
  const tensor part{{100000, 200}, {1, 0}, {64, 1}};  // columns of a row
  expect(!two(part, part, 64) && !two(part, part, -136) && two(part, part, 63) && two(part, part, 200), "columns");
  const tensor one{{100000, 6144}, {128, 1}};  // a head that many are to be
  expect(!two(q, one, 4096 + 128) && two(q, one, 4095), "a head of a slice");
  const tensor heads{{4, 1000 * 64}, {1000, 64}, {64, 1}}, slots{{1000, 64}, {4, 1000 * 64}, {64, 1}};
  expect(two(heads, slots, 0) && !two(heads, slots, 4000 * 64), "a transposed tensor");
  expect(!shares_itself(q.data(), 3) && !shares_itself(slots.data(), 3), "no tensor of these shares itself");
  const tensor window{{1000, 64}, {128, 1}};
  expect(shares_itself(window.data(), 2), "windows do");
  std::printf("ok\n");
}
