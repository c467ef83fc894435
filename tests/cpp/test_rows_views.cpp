// C++ host layer: the row operators over views — states inside wider rows, one mask for all rows, a selection whose memory is used again.  Values are worked
// out by hand.  Build + run: tests/test_cpp_rows.py.  Prints "ALL OK" and exits 0 on success.
#include <cmath>
#include <cstdio>

#include "../../host/arrow_gpu.hpp"

using namespace arrow_gpu;
static int failures = 0;
#define CHECK(cond)                                               \
  do {                                                            \
    if (!(cond)) {                                                \
      std::printf("FAIL %s:%d  %s\n", __FILE__, __LINE__, #cond); \
      failures++;                                                 \
    }                                                             \
  } while (0)

template <typename F> static bool throws(F f) {
  try {
    f();
  } catch (const ArrowErrorGPU&) {
    return true;
  }
  return false;
}

static void run(const DevicePtr& dev) {
  ArrowComputePipeline p(dev);
  {  // 3 rows of (old, new) x 2 pieces of 2 words: the old halves of rows 2, 0, 0 go into the new ones, in one allocation
    std::vector<uint32_t> held(24);
    for (uint32_t i = 0; i < 24; i++) held[i] = i;
    const auto buf = dev->create_gpu_buffer_with_data(held.data(), 24);
    const StateGPU before{buf, 3, 2, 8, 4, 32, 8, 0}, after{buf, 3, 2, 8, 4, 32, 8, 16};
    const auto parents = UInt32ArrayGPU::from_slice({2, 0, 0}, dev);
    take_rows_op({before}, parents, {after}, p);
    p.sync();
    auto raw = dev->retrive_data(buf, 96);
    std::vector<uint32_t> got(24);
    std::memcpy(got.data(), raw.data(), 96);
    CHECK((got == std::vector<uint32_t>{0, 1, 2, 3, 16, 17, 18, 19, 8, 9, 10, 11, 0, 1, 2, 3, 16, 17, 18, 19, 0, 1, 2, 3}));
    // pieces with a gap behind each: words 0 and 2 of every row, nothing for row 1
    const StateGPU gaps{buf, 3, 2, 4, 4, 32, 8, 0};
    const StateGPU dense{dev->create_gpu_buffer_with_data(std::vector<uint32_t>(6, 7).data(), 6), 3, 2, 4, 4};
    take_rows_op({gaps}, parents, {dense}, p, UInt32ArrayGPU::from_slice({1, 0, 5}, dev));
    p.sync();
    raw = dev->retrive_data(dense.data, 24);
    got.resize(6);
    std::memcpy(got.data(), raw.data(), 24);
    CHECK((got == std::vector<uint32_t>{16, 18, 7, 7, 0, 2}));
    CHECK(throws([&] { take_rows_op({before}, parents, {before}, p); }));
    CHECK(throws([&] { take_rows_op({StateGPU{buf, 3, 2, 8, 4, 32, 8, 24}}, parents, {dense}, p); }));       // 64 + 8 + 8 + 24 bytes
    CHECK(throws([&] { take_rows_op({StateGPU{buf, 3, 2, 4, 4, ~0ull, 8, 0}}, parents, {dense}, p); }));    // past 2^64
  }
  {  // one mask for both rows: tokens 1 and 3 of (0, ln 3, 9, 0) and (5, 0, 0, 0)
    const auto logits = RowsGPU::from_slice({0.0f, std::log(3.0f), 9.0f, 0.0f, 5.0f, 0.0f, 0.0f, 0.0f}, 1, 4, dev);
    std::vector<uint8_t> bits(8, 0);
    bits[0] = 10;
    const auto cum = Float32ArrayGPU::from_slice({std::log(0.6f), std::log(0.4f)}, dev);  // 0.6 x (3/4, 1/4) = 0.45, 0.15; 0.4 x 1/2 = 0.2 twice
    const auto first = select_beams_op(logits, 2, 4, p, cum, BooleanArrayGPU(dev->create_gpu_buffer_with_data(bits.data(), 8), dev, 4, std::nullopt));
    const auto padded = select_beams_op(logits, 2, 4, p, cum, BooleanArrayGPU(dev->create_gpu_buffer_with_data(bits.data(), 8), dev, 64, std::nullopt));
    p.sync();
    for (const auto* s : {&first, &padded}) {
      CHECK((s->parents.raw_values() == std::vector<uint32_t>{0, 1, 1, 0}) && (s->tokens.raw_values() == std::vector<uint32_t>{1, 1, 3, 3}));
      CHECK(std::fabs(s->scores.raw_values()[0] - std::log(0.45f)) < 1e-6f);
    }
    // into the first one's memory, without the mask: 9 and 5 win
    const auto again = select_beams_op(logits, 2, 4, p, cum, std::nullopt, std::nullopt, 0, &first);
    p.sync();
    CHECK(again.scores.data == first.scores.data && again.parents.data == first.parents.data && again.tokens.data == first.tokens.data && again.workspace == first.workspace);
    CHECK(first.tokens.raw_values()[0] == 2 && first.tokens.raw_values()[1] == 0 && first.parents.raw_values()[1] == 1);
    CHECK(throws([&] { select_beams_op(logits, 2, 3, p, cum, std::nullopt, std::nullopt, 0, &first); }));
    CHECK(throws([&] { select_beams_op(logits, 2, 4, p, first.scores, std::nullopt, std::nullopt, 0, &first); }));  // 4 scores for 2 rows
    CHECK(throws([&] { select_beams_op(logits, 1, 1, p, again.scores, std::nullopt, std::nullopt, 0, &first); }));
  }
}

int main() {
  DevicePtr dev;
  try {
    dev = GpuDevice::create(0);
  } catch (const ArrowErrorGPU& e) {
    std::printf("no device: %s\n", e.what());
    return 2;
  }
  run(dev);
  if (failures) return 1;
  std::printf("ALL OK\n");
  return 0;
}
