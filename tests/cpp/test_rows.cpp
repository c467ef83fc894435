// C++ host layer: the row operators (quantised caches, beam selection, states) through host/arrow_gpu.hpp → C ABI → HIP, one step of a search and
// what the calls refuse.  Values are worked out by hand.  Build + run: tests/test_cpp_rows.py.  Prints "ALL OK" and exits 0 on success.
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

static std::vector<float> read(const RowsGPU& r) {
  const auto raw = r.gpu_device->retrive_data(r.data, 4 * r.rows * r.heads * r.dim);
  std::vector<float> v(raw.size() / 4);
  std::memcpy(v.data(), raw.data(), raw.size());
  return v;
}
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
  {  // two rows of 2 heads x 8: whole numbers up to 127 come back exactly from 8 bits, 0..15 from 4
    std::vector<float> a(32), b(32);
    for (int i = 0; i < 32; i++) a[i] = (float)(i % 8 == 7 ? 127 : 3 * i - 40), b[i] = (float)((5 * i) % 16);
    for (int g = 0; g < 4; g++) b[8 * g] = 0.0f, b[8 * g + 1] = 15.0f;
    const std::vector<QuantisedRowsGPU> stores{QuantisedRowsGPU::empty(6, 2, 8, 8, AGPU_CODE_I8, dev), QuantisedRowsGPU::empty(6, 2, 8, 8, AGPU_CODE_I4, dev)};
    const auto slots = UInt32ArrayGPU::from_slice({4, 1}, dev);
    put_quantised_op(stores, {RowsGPU::from_slice(a, 2, 8, dev), RowsGPU::from_slice(b, 2, 8, dev)}, slots, p);
    const std::vector<RowsGPU> out{RowsGPU::empty(2, 2, 8, AGPU_ROW_F32, dev), RowsGPU::empty(2, 2, 8, AGPU_ROW_F32, dev)};
    take_quantised_op(stores, slots, out, p);
    p.sync();
    CHECK(read(out[0]) == a && read(out[1]) == b);
    // the same rows through a page table: pages of 3 rows, page 1 = slots 3..5, page 0 = slots 0..2; positions 1 (slot 4) and 4 (slot 1)
    const PageMap pages{UInt32ArrayGPU::from_slice({1, 0}, dev), UInt32ArrayGPU::from_slice({0, 4}, dev), 2, 3, UInt32ArrayGPU::from_slice({1}, dev)};
    const std::vector<RowsGPU> four{RowsGPU::empty(4, 2, 8, AGPU_ROW_F32, dev), RowsGPU::empty(4, 2, 8, AGPU_ROW_F32, dev)};
    take_quantised_op(stores, pages, four, p);
    p.sync();
    const auto r = read(four[0]);
    CHECK(std::vector<float>(r.begin(), r.begin() + 16) == std::vector<float>(a.begin(), a.begin() + 16));
    CHECK(std::vector<float>(r.begin() + 48, r.end()) == std::vector<float>(a.begin() + 16, a.end()));
    for (int i = 16; i < 48; i++) CHECK(r[i] == 0.0f);
    put_quantised_op(stores, four, pages, p);  // and back again: nothing changes
    take_quantised_op(stores, slots, out, p);
    p.sync();
    CHECK(read(out[0]) == a);
    take_quantised_op(stores, UInt32ArrayGPU::from_slice({4, 6}, dev), out, p);  // slot 6 of 6
    CHECK(throws([&] { p.sync(); }));
    CHECK(read(out[0])[0] == a[0] && read(out[0])[16] == 0.0f);
    CHECK(throws([&] { take_quantised_op(stores, slots, {out[0]}, p); }));
    CHECK(throws([&] { take_quantised_op(stores, UInt32ArrayGPU::from_slice({1}, dev), out, p); }));
  }
  {  // 2 beams x 4 tokens: log-softmax of (0, ln 2, ln 4, 0) = ln(1/8, 2/8, 4/8, 1/8), of (0, 0, 0, 0) = ln 1/4 each
    const float l2 = std::log(2.0f), l4 = std::log(4.0f);
    const auto logits = RowsGPU::from_slice({0.0f, l2, l4, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, 1, 4, dev);
    const auto sel = select_beams_op(logits, 2, 4, p, Float32ArrayGPU::from_slice({std::log(0.5f), std::log(0.6f)}, dev));
    // 0.5 · 1/2 = 0.25, then 0.6 · 1/4 = 0.15 three times in token order (0.5 · 2/8 = 0.125 comes behind the fourth)
    p.sync();
    CHECK((sel.parents.raw_values() == std::vector<uint32_t>{0, 1, 1, 1}));
    CHECK((sel.tokens.raw_values() == std::vector<uint32_t>{2, 0, 1, 2}));
    const auto s = sel.scores.raw_values();
    CHECK(std::fabs(s[0] - std::log(0.25f)) < 1e-6f && std::fabs(s[3] - std::log(0.15f)) < 1e-6f);
    // a finished beam, and a mask that leaves token 3
    std::vector<uint8_t> bits(16, 0);
    bits[0] = 8, bits[8] = 8;
    const auto allowed = BooleanArrayGPU(dev->create_gpu_buffer_with_data(bits.data(), bits.size()), dev, 128, std::nullopt);
    const auto done = BooleanArrayGPU::from_slice({false, true}, dev);
    const auto masked = select_beams_op(logits, 2, 3, p, Float32ArrayGPU::from_slice({-1.0f, -0.5f}, dev), allowed, done, 1);
    p.sync();
    CHECK((masked.parents.raw_values() == std::vector<uint32_t>{1, 0, 0}) && (masked.tokens.raw_values() == std::vector<uint32_t>{1, 3, 0}));
    CHECK((masked.scores.raw_values() == std::vector<float>{-0.5f, -1.0f, -INFINITY}));
    // the states by the parents: rows of 2 pieces of 3 positions of 4 bytes
    std::vector<uint32_t> held(12);
    for (uint32_t i = 0; i < 12; i++) held[i] = 100 + i;
    const std::vector<StateGPU> from{{dev->create_gpu_buffer_with_data(held.data(), 12), 2, 2, 12, 4}};
    const std::vector<uint32_t> nine(24, 9);
    const std::vector<StateGPU> to{{dev->create_gpu_buffer_with_data(nine.data(), 24), 4, 2, 12, 4}};
    take_rows_op(from, sel.parents, to, p, UInt32ArrayGPU::from_slice({3, 2, 0, 1}, dev));
    p.sync();
    const auto raw = dev->retrive_data(to[0].data, 96);
    std::vector<uint32_t> got(24);
    std::memcpy(got.data(), raw.data(), 96);
    CHECK((got == std::vector<uint32_t>{100, 101, 102, 103, 104, 105, 106, 107, 9, 109, 110, 9, 9, 9, 9, 9, 9, 9, 106, 9, 9, 109, 9, 9}));
    CHECK(throws([&] { take_rows_op(to, sel.parents, to, p); }));  // in place
    CHECK(throws([&] { select_beams_op(logits, 3, 1, p); }) && throws([&] { select_beams_op(logits, 2, 65, p); }) && throws([&] { select_beams_op(logits, 2, 9, p); }));
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
