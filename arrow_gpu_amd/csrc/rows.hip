// rows.hip — take / put of whole rows: a cache quantised as it is written and read back, states reordered by an index column.
//
// Arithmetic of the codes (include/arrow_gpu.h agpu_quantised_rows).  The quotients top / span and span / top are one IEEE f32 division a
// group; a code is rint(x · inv) with the product rounded ONCE: fma(x, inv, 1.5 · 2^23) has the whole number in its low mantissa bits, ties to
// even, |x · inv| <= 127.00002.  The e4m3 code is made from the product in f32, which is what the conversion instruction takes.
#include "common.hpp"
#include "row_address.hpp"

namespace {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// ---------------------------------------------------------------- codes
template <int CODE> struct Top;
template <> struct Top<AGPU_CODE_I8> { static constexpr float v = 127.0f; };
template <> struct Top<AGPU_CODE_I4> { static constexpr float v = 15.0f; };
template <> struct Top<AGPU_CODE_E4M3> { static constexpr float v = 448.0f; };

struct Factors {
  float scale, inv, lo;
};
// span: max |x| or max − min, not finite where the group holds a NaN or an infinity
template <int CODE>
__device__ __forceinline__ Factors factors(float span, float lo) {
  constexpr float top = Top<CODE>::v;
  if (!(span < __builtin_inff())) return {__builtin_nanf(""), 0.0f, lo};
  if (span < top * 0x1p-126f) return {0.0f, 0.0f, lo};  // span / top would be subnormal and top / span could overflow
  // span / top, rounded once: the remainder of span · (1 / top) is exact and corrects it (compared with the division for all 2^23 mantissas)
  constexpr float r = 1.0f / top;
  const float q = span * r;
  return {__builtin_fmaf(__builtin_fmaf(-q, top, span), r, q), top / span, lo};
}
__device__ __forceinline__ uint32_t whole(float x, float inv) {  // low byte: the code in two's complement
  return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, inv, 0x1.8p23f));
}

// of three, a NaN if there is one
__device__ __forceinline__ float maximum_of(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float maximum_of_abs(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float minimum_of(float a, float b, float c) {
  float r;
  asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

struct QuantCol {
  void* x;
  uint64_t row_stride, head_stride;
  uint8_t* codes;
  float* scales;
  uint64_t n_slots;
};
struct QuantShape {
  uint32_t heads, dim, group, groups_per_head, groups_per_row;
};

// ---------------------------------------------------------------- 16 bytes of values a lane
// Both ways stream: 16-byte accesses on the rows' side (two of f32 a lane, 32 bytes apart, would write parts of lines: 468 us instead of 201 for two
// columns of 131072 rows of 4 bits as f32), 2 to 8 bytes on the codes'.  A group is `lanes` neighbouring lanes (a power of two, those
// past the group's end idle), its span found with data-parallel moves inside the wave.  A block takes whole rows, looks their slots up once and
// keeps them in LDS: a search of the sequence through memory costs microseconds, so it is shared by up to 8 passes of the block (16 passes: 131072
// rows of 4 bits in 138 us instead of 127).
// What bounds it is memory (least and average of 100 launches): two columns of 16384 rows of 8 x 128 bf16 go to e4m3 in 17.1 and 19.8 us and come back in 16.1 and
// 18.1 (102 MB each: 6.0 to 5.2 TB/s, 6.3 to 5.6; a copy of as many bytes takes 19), ragged e4m3 rows of 4 x 96 come back as f16 in 30.4 and 32.0 us (181 MB, 6.0 to
// 5.7 TB/s), two columns of 131072 rows of 4 bits as bf16 in 126.7 and 129.6 us (705 MB, 5.6 to 5.4 TB/s; a u8 -> f32 cast of as many bytes 112).  A token's rows
// take 2.3 and 2.7 us a call, that is one launch.
constexpr int MAX_COLS = 8, MAX_ROWS = 256;
struct QuantCols {
  QuantCol c[MAX_COLS];
};
struct FastShape {
  uint32_t group, groups_per_row, lanes, log_lanes, rows;  // rows of a block
  bool dense;                                                  // a row's heads follow each other
  Divide by_row, by_head;                                      // groups a row, groups a head
};

// Vectors of `many` values, from any element (any byte of the codes) on
template <typename T> struct Wide;
template <> struct Wide<float> {
  static constexpr int many = 4;
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Wide<f16_t> {
  static constexpr int many = 8;
  typedef f16_t type __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Wide<bf16_t> {
  static constexpr int many = 8;
  typedef bf16_t type __attribute__((ext_vector_type(8), aligned(2)));
};
typedef uint16_t u16_at_1 __attribute__((aligned(1)));
typedef uint32_t u32_at_1 __attribute__((aligned(1)));
typedef uint32_t u32x2_at_1 __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x2_at_4 __attribute__((ext_vector_type(2), aligned(4)));

template <int CTRL>
__device__ __forceinline__ float moved(float x) {  // another lane's of the row of 16
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
// f over the `lanes` lanes of a group: neighbour, pair, then mirrored halves — after the steps before them all lanes of a half agree
template <typename F>
__device__ __forceinline__ float over_group(float x, uint32_t lanes, F f) {
  if (lanes > 1) x = f(x, moved<0xB1>(x));   // quad_perm 1 0 3 2
  if (lanes > 2) x = f(x, moved<0x4E>(x));   // quad_perm 2 3 0 1
  if (lanes > 4) x = f(x, moved<0x141>(x));  // row_half_mirror
  if (lanes > 8) x = f(x, moved<0x140>(x));  // row_mirror
  if (lanes > 16) x = f(x, __shfl_xor(x, 16));
  if (lanes > 32) x = f(x, __shfl_xor(x, 32));
  return x;
}

// a row of the block: the number of its first group in the cache (ROW_NONE, ROW_BAD), and where its values begin (from the column's: a pointer out of LDS
// would be one into any memory, and its accesses the slower ones)
struct BlockRow {
  uint64_t at, x;
};
__device__ __forceinline__ uint32_t block_rows(const QuantCol& c, const FastShape& q, const RowAddr& addr, uint64_t n, BlockRow* held, uint32_t* flags) {
  const uint64_t row0 = (uint64_t)blockIdx.x * q.rows;
  const uint32_t rows = (uint32_t)(n - row0 < q.rows ? n - row0 : q.rows);
  if (threadIdx.x < rows) {
    const uint64_t row = row0 + threadIdx.x, s = row_slot(addr, row, c.n_slots);
    held[threadIdx.x] = {s < ROW_BAD ? s * q.groups_per_row : s, row * c.row_stride};
    if (s == ROW_BAD) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
  }
  __syncthreads();
  return rows;
}
// what a lane has at a time: W values of one group, from value `from` on; the last lane of a group that is no multiple of W has the group's last W (some of
// its neighbour's too: they get the same codes)
struct Unit {
  uint32_t row, in_row, from;
  bool idle;  // past the group's end
};
template <int W>
__device__ __forceinline__ Unit unit_of(uint32_t i, const FastShape& q) {
  const uint32_t g = i >> q.log_lanes, row = g / q.by_row, from = (i & (q.lanes - 1)) * W;
  return {row, g - row * q.groups_per_row, from + W <= q.group ? from : q.group - W, from >= q.group};
}
__device__ __forceinline__ uint64_t value_offset(const Unit& u, const QuantCol& c, const FastShape& q) {
  if (q.dense) return u.in_row * q.group + u.from;
  const uint32_t head = u.in_row / q.by_head;
  return head * c.head_stride + (u.in_row - head * q.by_head.d) * q.group + u.from;
}

template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void put_wide_kernel(QuantCols cols, FastShape q, RowAddr addr, uint64_t n, uint32_t* flags) {
  typedef typename Wide<T>::type Vector;
  constexpr int W = Wide<T>::many;
  __shared__ BlockRow held[MAX_ROWS];
  const QuantCol& c = cols.c[blockIdx.y];  // (one load of a lane in flight: two or four do not pay, 18.2 -> 18.9 us of 2 x 16384 rows)
  const uint32_t total = (block_rows(c, q, addr, n, held, flags) * q.groups_per_row) << q.log_lanes;
  for (uint32_t i = threadIdx.x; i < total; i += AGPU_BLOCK) {
    const Unit t = unit_of<W>(i, q);
    const BlockRow row = held[t.row];
    const bool live = !t.idle && row.at < ROW_BAD;
    float v[W] = {};
    if (live) {
      const Vector w = *reinterpret_cast<const Vector*>(static_cast<const T*>(c.x) + row.x + value_offset(t, c, q));
#pragma unroll
      for (int j = 0; j < W; j++) v[j] = (float)w[j];
    }
    // the largest magnitude, or the lowest and the highest value; a NaN stays
    float span, lo = 0.0f;
    if (CODE == AGPU_CODE_I4) {
      float l = live ? v[0] : __builtin_inff(), h = live ? v[0] : -__builtin_inff();
      if (live) {
#pragma unroll
        for (int j = 1; j < W; j += 2) l = minimum_of(l, v[j], v[j + 1 < W ? j + 1 : j]), h = maximum_of(h, v[j], v[j + 1 < W ? j + 1 : j]);
      }
      lo = over_group(l, q.lanes, [](float a, float b) { return minimum_of(a, b, b); });
      span = over_group(h, q.lanes, [](float a, float b) { return maximum_of(a, b, b); }) - lo;
    } else {
      float most = 0.0f;
#pragma unroll
      for (int j = 0; j < W; j += 2) most = maximum_of_abs(most, v[j], v[j + 1]);
      span = over_group(most, q.lanes, [](float a, float b) { return maximum_of(a, b, b); });
    }
    const Factors f = factors<CODE>(span, lo);
    if (!live) continue;
    const uint64_t at = row.at + t.in_row;
    if (CODE == AGPU_CODE_I4) {
      if (t.from == 0) reinterpret_cast<f32x2_at_4*>(c.scales)[at] = f32x2_at_4{f.scale, f.lo};
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < W; j++) w |= (whole(v[j] - f.lo, f.inv) & 15) << 4 * j;
      uint8_t* to = c.codes + at * (q.group / 2) + t.from / 2;
      if constexpr (W == 8) *reinterpret_cast<u32_at_1*>(to) = w;
      else *reinterpret_cast<u16_at_1*>(to) = (uint16_t)w;
    } else {
      if (t.from == 0) c.scales[at] = f.scale;
      u32x2_at_1 w;
#pragma unroll
      for (int h = 0; h < W / 4; h++) {
        if (CODE == AGPU_CODE_I8) {
          w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(whole(v[4 * h + 3], f.inv), whole(v[4 * h + 2], f.inv), 0x0C0C0400u),
                                       __builtin_amdgcn_perm(whole(v[4 * h + 1], f.inv), whole(v[4 * h], f.inv), 0x0C0C0400u), 0x05040100u);
        } else {
          const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * f.inv, v[4 * h + 1] * f.inv, 0, false);
          w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * f.inv, v[4 * h + 3] * f.inv, low, true);
        }
      }
      uint8_t* to = c.codes + at * q.group + t.from;
      if constexpr (W == 8) *reinterpret_cast<u32x2_at_1*>(to) = w;
      else *reinterpret_cast<u32_at_1*>(to) = w.x;
    }
  }
}

constexpr int TAKE_UNROLL = 8;  // all of a block's passes in flight: 131072 rows of 4 bits 127 us, of four at a time 132

template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void take_wide_kernel(QuantCols cols, FastShape q, RowAddr addr, uint64_t n, uint32_t* flags) {
  typedef typename Wide<T>::type Vector;
  constexpr int W = Wide<T>::many;
  __shared__ BlockRow held[MAX_ROWS];
  const QuantCol& c = cols.c[blockIdx.y];
  const uint32_t total = (block_rows(c, q, addr, n, held, flags) * q.groups_per_row) << q.log_lanes;
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += AGPU_BLOCK * TAKE_UNROLL) {
    uint64_t to[TAKE_UNROLL];  // from the column's first value
    u32x2 w[TAKE_UNROLL];
    f32x2_at_4 f[TAKE_UNROLL];
#pragma unroll
    for (int u = 0; u < TAKE_UNROLL; u++) {
      const uint32_t i = i0 + u * AGPU_BLOCK;
      to[u] = ROW_NONE;
      w[u] = u32x2{0, 0}, f[u] = f32x2_at_4{0.0f, 0.0f};  // out of range: zeros
      const Unit t = unit_of<W>(i, q);
      if (i >= total || t.idle) continue;
      const BlockRow row = held[t.row];
      if (row.at == ROW_NONE) continue;
      to[u] = row.x + value_offset(t, c, q);
      if (row.at == ROW_BAD) continue;
      const uint64_t at = row.at + t.in_row;
      if (CODE == AGPU_CODE_I4) {
        f[u] = reinterpret_cast<const f32x2_at_4*>(c.scales)[at];
        const uint8_t* from = c.codes + at * (q.group / 2) + t.from / 2;
        if constexpr (W == 8) w[u].x = *reinterpret_cast<const u32_at_1*>(from);
        else w[u].x = *reinterpret_cast<const u16_at_1*>(from);
      } else {
        f[u].x = c.scales[at];
        const uint8_t* from = c.codes + at * q.group + t.from;
        if constexpr (W == 8) w[u] = *reinterpret_cast<const u32x2_at_1*>(from);
        else w[u].x = *reinterpret_cast<const u32_at_1*>(from);
      }
    }
#pragma unroll
    for (int u = 0; u < TAKE_UNROLL; u++) {
      if (to[u] == ROW_NONE) continue;
      Vector o;
      if (CODE == AGPU_CODE_I4) {
        const uint32_t even = w[u].x & 0x0F0F0F0Fu, odd = w[u].x >> 4 & 0x0F0F0F0Fu;  // a byte each: the conversion takes them from where they are
#pragma unroll
        for (int j = 0; j < W / 2; j++) {
          o[2 * j] = (T)__builtin_fmaf((float)(even >> 8 * j & 255), f[u].x, f[u].y);
          o[2 * j + 1] = (T)__builtin_fmaf((float)(odd >> 8 * j & 255), f[u].x, f[u].y);
        }
      } else {
#pragma unroll
        for (int h = 0; h < W / 4; h++) {
          const uint32_t b = w[u][h];
          if (CODE == AGPU_CODE_E4M3) {
            const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(b, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(b, true);
            o[4 * h] = (T)(low[0] * f[u].x), o[4 * h + 1] = (T)(low[1] * f[u].x), o[4 * h + 2] = (T)(high[0] * f[u].x), o[4 * h + 3] = (T)(high[1] * f[u].x);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) o[4 * h + j] = (T)((float)(int8_t)(b >> 8 * j) * f[u].x);
          }
        }
      }
      // past the caches: nobody reads the rows in this call (ragged e4m3 rows 30.5 us, through the caches 42)
      __builtin_nontemporal_store(o, reinterpret_cast<Vector*>(static_cast<T*>(c.x) + to[u]));
    }
  }
}

// ---------------------------------------------------------------- a value a lane at a time: groups below 16 bytes and above 64 times that
// A group is `lanes` neighbouring lanes, at most a wave.  Bound by its narrow accesses and a slot's look-up for each group: 2^24 bf16 values in groups of
// 1024 go to 8 bits in 26.5 us and come back in 18.1 on average, of 576 in 30.4 and 20.7 (of 512, in the form above: 13 and 11).
template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void put_group_kernel(QuantCol c, QuantShape q, RowAddr addr, uint64_t n_groups, uint32_t lanes, uint32_t* flags) {
  const uint32_t lane = threadIdx.x % lanes, held = AGPU_BLOCK / lanes;
  const uint64_t step = (uint64_t)gridDim.x * held;
  for (uint64_t g = (uint64_t)blockIdx.x * held + threadIdx.x / lanes; g < n_groups; g += step) {  // (the lanes of a group go together)
    const uint64_t row = g / q.groups_per_row;
    const uint32_t in_row = (uint32_t)(g - row * q.groups_per_row), head = in_row / q.groups_per_head;
    const uint64_t slot = row_slot(addr, row, c.n_slots);
    if (slot >= ROW_BAD) {
      if (slot == ROW_BAD && lane == 0) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
      continue;
    }
    const T* x = static_cast<const T*>(c.x) + row * c.row_stride + head * c.head_stride + (in_row - head * q.groups_per_head) * q.group;
    float lo = __builtin_inff(), hi = -__builtin_inff();
    uint32_t bad = 0;
    for (uint32_t i = lane; i < q.group; i += lanes) {
      const float v = (float)x[i];
      bad |= !(__builtin_fabsf(v) < __builtin_inff());
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
    }
    for (uint32_t d = lanes / 2; d; d >>= 1) {
      lo = fminf(lo, __shfl_xor(lo, d));
      hi = fmaxf(hi, __shfl_xor(hi, d));
      bad |= __shfl_xor(bad, d);
    }
    const Factors f = factors<CODE>(bad ? __builtin_nanf("") : CODE == AGPU_CODE_I4 ? hi - lo : fmaxf(hi, -lo), lo);
    const uint64_t at = slot * q.groups_per_row + in_row;
    if (CODE == AGPU_CODE_I4) {
      if (lane == 0) c.scales[2 * at] = f.scale, c.scales[2 * at + 1] = f.lo;
      for (uint32_t i = lane; i < q.group / 2; i += lanes)
        c.codes[at * (q.group / 2) + i] = (uint8_t)((whole((float)x[2 * i] - f.lo, f.inv) & 15) | (whole((float)x[2 * i + 1] - f.lo, f.inv) & 15) << 4);
    } else {
      if (lane == 0) c.scales[at] = f.scale;
      for (uint32_t i = lane; i < q.group; i += lanes) {
        const float v = (float)x[i];
        c.codes[at * q.group + i] = CODE == AGPU_CODE_I8 ? (uint8_t)whole(v, f.inv)
                                                         : (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v * f.inv, 0.0f, 0, false);
      }
    }
  }
}

template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void take_group_kernel(QuantCol c, QuantShape q, RowAddr addr, uint64_t n_groups, uint32_t lanes, uint32_t* flags) {
  const uint32_t lane = threadIdx.x % lanes, held = AGPU_BLOCK / lanes;
  const uint64_t step = (uint64_t)gridDim.x * held;
  for (uint64_t g = (uint64_t)blockIdx.x * held + threadIdx.x / lanes; g < n_groups; g += step) {
    const uint64_t row = g / q.groups_per_row;
    const uint32_t in_row = (uint32_t)(g - row * q.groups_per_row), head = in_row / q.groups_per_head;
    const uint64_t slot = row_slot(addr, row, c.n_slots);
    if (slot == ROW_NONE) continue;
    const bool ok = slot != ROW_BAD;
    if (!ok && lane == 0) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
    T* x = static_cast<T*>(c.x) + row * c.row_stride + head * c.head_stride + (in_row - head * q.groups_per_head) * q.group;
    const uint64_t at = slot * q.groups_per_row + in_row;
    const float scale = !ok ? 0.0f : c.scales[CODE == AGPU_CODE_I4 ? 2 * at : at], lo = ok && CODE == AGPU_CODE_I4 ? c.scales[2 * at + 1] : 0.0f;
    for (uint32_t i = lane; i < q.group; i += lanes) {
      float v = 0.0f;
      if (ok && CODE == AGPU_CODE_I4) v = __builtin_fmaf((float)((c.codes[(at * q.group + i) / 2] >> (4 * (i & 1))) & 15), scale, lo);
      else if (ok && CODE == AGPU_CODE_I8) v = (float)(int8_t)c.codes[at * q.group + i] * scale;
      else if (ok) v = __builtin_amdgcn_cvt_f32_fp8(c.codes[at * q.group + i], 0) * scale;
      x[i] = (T)v;
    }
  }
}

// ---------------------------------------------------------------- host: checks and dispatch
// where: the slot column, or the page map's three columns
agpu_status check_columns(int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, uint64_t n, bool writes_rows, std::initializer_list<Places> where) {
  Places places[3 * 64 + 3];
  uint32_t count = 0;
  if (writes_rows)
    for (const Places& w : where)
      if (w.at && w.size) places[count++] = w;
  for (int32_t k = 0; k < n_cols; k++) {
    const agpu_quantised_rows& s = stores[k];
    const agpu_rows& r = rows[k];
    AGPU_REQUIRE(r.row_type >= AGPU_ROW_F32 && r.row_type <= AGPU_ROW_BF16, AGPU_ERR_ARG, "row type");
    AGPU_REQUIRE(s.code >= AGPU_CODE_I8 && s.code <= AGPU_CODE_E4M3, AGPU_ERR_ARG, "code type");
    AGPU_REQUIRE(s.heads > 0 && s.dim > 0 && (uint64_t)s.heads * s.dim <= (1u << 30), AGPU_ERR_SHAPE, "1 <= heads * dim <= 2^30");
    AGPU_REQUIRE(s.group > 0 && s.group <= 65536 && s.dim % s.group == 0, AGPU_ERR_SHAPE, "group divides dim, 1 <= group <= 65536");
    AGPU_REQUIRE(s.code != AGPU_CODE_I4 || s.group % 2 == 0, AGPU_ERR_SHAPE, "4-bit codes: an even group");
    AGPU_REQUIRE(s.n_slots <= (1ull << 32), AGPU_ERR_SHAPE, "n_slots <= 2^32");
    AGPU_REQUIRE(n * s.heads * s.dim < (1ull << 48), AGPU_ERR_SHAPE, "less than 2^48 values a column");
    AGPU_REQUIRE(r.data && s.codes && s.scales, AGPU_ERR_ARG, "null pointer");
    AGPU_REQUIRE(aligned_to(r.data, r.row_type == AGPU_ROW_F32 ? 4 : 2) && aligned_to(s.scales, 4), AGPU_ERR_SHAPE, "alignment");
    if (writes_rows) {
      AGPU_REQUIRE(disjoint(n, r.row_stride, s.heads, r.head_stride, s.dim), AGPU_ERR_SHAPE, "rows that are written may not overlap");
      const uint64_t item = r.row_type == AGPU_ROW_F32 ? 4 : 2;
      uint64_t bytes;
      AGPU_REQUIRE(r.row_stride < (1ull << 61) && r.head_stride < (1ull << 61) &&
                       extent(n, r.row_stride * item, s.heads, r.head_stride * item, s.dim * item, &bytes), AGPU_ERR_SHAPE, "rows past the address space");
      places[count++] = {reinterpret_cast<uintptr_t>(r.data), n, r.row_stride * item, s.heads, r.head_stride * item, s.dim * item, true, 2 * k};
    }
    const uint64_t values = s.n_slots * s.heads * s.dim, pair = s.code == AGPU_CODE_I4 ? 2 : 1;
    if (s.n_slots == 0) continue;
    places[count++] = {reinterpret_cast<uintptr_t>(s.codes), 1, 0, 1, 0, values / pair, !writes_rows, 2 * k + 1};
    places[count++] = {reinterpret_cast<uintptr_t>(s.scales), 1, 0, 1, 0, values / s.group * 4 * pair, !writes_rows, 2 * k + 1};
  }
  uint32_t x, y;
  if (overlapping(places, count, &x, &y)) {
    AGPU_REQUIRE(writes_rows, AGPU_ERR_ARG, "two columns into one cache");
    AGPU_REQUIRE(places[x].written && places[y].written, AGPU_ERR_ARG, "rows that are written overlap a cache or the slots");
    AGPU_REQUIRE(false, AGPU_ERR_ARG, "the rows of two columns overlap");
  }
  return AGPU_OK;
}

// 16 bytes of values a lane: a group that has them and fits a wave (2^24 bf16 values in groups of 100 to 8 bits: 16 us, a value a lane at a time 64)
bool is_wide(uint32_t group, uint32_t many) { return group >= many && group <= 64 * many; }

// Rows of a block: 8 passes of its lanes, fewer where that would leave less than 2048 blocks (8 a CU)
FastShape fast_shape(const QuantShape& q, uint32_t many, uint64_t n, uint32_t n_cols) {
  FastShape f = {};
  f.group = q.group, f.groups_per_row = q.groups_per_row;
  while (many << f.log_lanes < q.group) f.log_lanes++;
  f.lanes = 1u << f.log_lanes;
  const uint64_t row_lanes = (uint64_t)q.groups_per_row << f.log_lanes;
  uint64_t rows = 8 * AGPU_BLOCK / row_lanes;
  if (rows * 2048 > n * n_cols) rows = n * n_cols / 2048;
  if (rows * row_lanes < AGPU_BLOCK) rows = AGPU_BLOCK / row_lanes;
  if (rows < n >> 23) rows = (n + (1u << 23) - 1) >> 23;  // a launch has less than 2^32 threads
  f.rows = (uint32_t)(rows < 1 ? 1 : rows > MAX_ROWS ? MAX_ROWS : rows);
  f.by_row = divide_by(q.groups_per_row), f.by_head = divide_by(q.groups_per_head);
  return f;
}

template <typename T, int CODE>
void launch_code(agpu_pipeline* p, bool put, const QuantCols& cols, uint32_t n_cols, const QuantShape& q, const RowAddr& addr, uint64_t n) {
  if (is_wide(q.group, Wide<T>::many)) {
    FastShape f = fast_shape(q, Wide<T>::many, n, n_cols);
    f.dense = true;
    for (uint32_t k = 0; k < n_cols; k++) f.dense = f.dense && (q.heads == 1 || cols.c[k].head_stride == q.dim);
    const dim3 grid((uint32_t)((n + f.rows - 1) / f.rows), n_cols);
    if (put) hipLaunchKernelGGL((put_wide_kernel<T, CODE>), grid, dim3(AGPU_BLOCK), 0, p->stream, cols, f, addr, n, p->flags);
    else hipLaunchKernelGGL((take_wide_kernel<T, CODE>), grid, dim3(AGPU_BLOCK), 0, p->stream, cols, f, addr, n, p->flags);
    return;
  }
  for (uint32_t k = 0; k < n_cols; k++) {
    uint32_t lanes = 1;
    while (lanes < 64 && lanes < q.group) lanes *= 2;
    const uint64_t n_groups = n * q.groups_per_row, blocks = (n_groups + AGPU_BLOCK / lanes - 1) / (AGPU_BLOCK / lanes);
    const int grid = (int)(blocks > (1u << 20) ? (1u << 20) : blocks);
    if (put) hipLaunchKernelGGL((put_group_kernel<T, CODE>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, cols.c[k], q, addr, n_groups, lanes, p->flags);
    else hipLaunchKernelGGL((take_group_kernel<T, CODE>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, cols.c[k], q, addr, n_groups, lanes, p->flags);
  }
}
template <typename T>
void launch_type(agpu_pipeline* p, bool put, int code, const QuantCols& cols, uint32_t n_cols, const QuantShape& q, const RowAddr& addr, uint64_t n) {
  switch (code) {
    case AGPU_CODE_I8: return launch_code<T, AGPU_CODE_I8>(p, put, cols, n_cols, q, addr, n);
    case AGPU_CODE_I4: return launch_code<T, AGPU_CODE_I4>(p, put, cols, n_cols, q, addr, n);
    default: return launch_code<T, AGPU_CODE_E4M3>(p, put, cols, n_cols, q, addr, n);
  }
}

agpu_status quantised(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const RowAddr& addr,
                      uint64_t n, const char* name) {
  AGPU_BIND_AS(p, name);
  if (n == 0) return AGPU_OK;
  // neighbouring columns of one kind go into one launch
  for (int32_t k = 0; k < n_cols;) {
    const agpu_quantised_rows& s = stores[k];
    const int type = rows[k].row_type;
    const QuantShape q = {s.heads, s.dim, s.group, s.dim / s.group, s.heads * (s.dim / s.group)};
    QuantCols cols;
    uint32_t m = 0;
    for (; k < n_cols && m < MAX_COLS; k++, m++) {
      const agpu_quantised_rows& o = stores[k];
      const agpu_rows& r = rows[k];
      if (o.heads != s.heads || o.dim != s.dim || o.group != s.group || o.code != s.code || r.row_type != type) break;
      cols.c[m] = {r.data, r.row_stride, r.head_stride, static_cast<uint8_t*>(o.codes), o.scales, o.n_slots};
    }
    if (type == AGPU_ROW_F32) launch_type<float>(p, put, s.code, cols, m, q, addr, n);
    else if (type == AGPU_ROW_F16) launch_type<f16_t>(p, put, s.code, cols, m, q, addr, n);
    else launch_type<bf16_t>(p, put, s.code, cols, m, q, addr, n);
    AGPU_LAUNCH_CHECK();
  }
  return AGPU_OK;
}

agpu_status quantised_slots(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const uint32_t* slots,
                            uint64_t n, const char* name) {
  AGPU_REQUIRE(n_cols >= 0 && n_cols <= 64, AGPU_ERR_ARG, "0 <= n_cols <= 64");
  RowAddr a = {};
  if (n_cols == 0 || n == 0) return quantised(p, put, 0, stores, rows, a, 0, name);
  AGPU_REQUIRE(stores && rows && slots, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(n < (1ull << 31), AGPU_ERR_SHAPE, "n < 2^31");
  AGPU_REQUIRE(aligned_to(slots, 4), AGPU_ERR_SHAPE, "alignment");
  const agpu_status st = check_columns(n_cols, stores, rows, n, !put, {{reinterpret_cast<uintptr_t>(slots), 1, 0, 1, 0, 4 * n, false, -1}});
  if (st != AGPU_OK) return st;
  a.slots = slots;
  return quantised(p, put, n_cols, stores, rows, a, n, name);
}

agpu_status quantised_pages(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const agpu_page_map* m,
                            uint64_t n, const char* name) {
  AGPU_REQUIRE(n_cols >= 0 && n_cols <= 64, AGPU_ERR_ARG, "0 <= n_cols <= 64");
  if (n_cols == 0 || n == 0) return quantised(p, put, 0, stores, rows, RowAddr{}, 0, name);
  AGPU_REQUIRE(stores && rows && m && m->offsets, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(n < (1ull << 31), AGPU_ERR_SHAPE, "n < 2^31");
  AGPU_REQUIRE(m->n_seqs > 0 && m->n_seqs < (1u << 31) && m->page_rows > 0, AGPU_ERR_SHAPE, "1 <= n_seqs < 2^31, page_rows >= 1");
  AGPU_REQUIRE(m->max_pages == 0 || m->tables, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(aligned_to(m->tables, 4) && aligned_to(m->offsets, 4) && aligned_to(m->first, 4), AGPU_ERR_SHAPE, "alignment");
  uint64_t tables;
  AGPU_REQUIRE(m->table_stride < (1ull << 61) && extent(m->n_seqs, 4 * m->table_stride, 1, 0, 4ull * m->max_pages, &tables), AGPU_ERR_SHAPE, "page tables past the address space");
  const agpu_status st = check_columns(n_cols, stores, rows, n, !put, {{reinterpret_cast<uintptr_t>(m->tables), m->n_seqs, 4 * m->table_stride, 1, 0, 4ull * m->max_pages, false, -1},
                                                                       {reinterpret_cast<uintptr_t>(m->offsets), 1, 0, 1, 0, 4ull * m->n_seqs + 4, false, -1},
                                                                       {reinterpret_cast<uintptr_t>(m->first), 1, 0, 1, 0, 4ull * m->n_seqs, false, -1}});
  if (st != AGPU_OK) return st;
  const RowAddr a = {nullptr, m->tables, m->table_stride, m->offsets, m->first, m->n_seqs, m->max_pages, m->page_rows};
  return quantised(p, put, n_cols, stores, rows, a, n, name);
}

// ---------------------------------------------------------------- take_rows
// A copy with one indirection: lanes run over the states' accesses of 16 bytes in the order of the destination, two of a lane in flight, all states in
// one launch (blockIdx.y).  Accesses begin at any byte; the last of a piece that is no multiple of 16 (or of what a length leaves) is the 16 bytes before
// its end, some of them its neighbour's too, the same.  Bound by memory: 904 MB in 146.9 us at least, 151.9 on average of 100 launches, 6.2 and 6.0 TB/s,
// where a copy of as many bytes reaches 6.6 (one or four of a lane in flight: 151 and 147 at least, of a short row's 3.6 and 4.8 instead of 3.5); 64 rows of
// 4000001 f32, no row on 16 bytes, in 349 us, 5.9 TB/s.
constexpr int MAX_STATES = 8, ROWS_UNROLL = 2;
struct State {
  const char* src;
  char* dst;
  uint64_t src_row_stride, src_piece_stride, dst_row_stride, dst_piece_stride, position_bytes;
  uint32_t n_vecs, vecs_per_row, piece_bytes;
  Divide by_row, by_piece;
};
struct States {
  State s[MAX_STATES];
};
typedef uint32_t u32x4_at_1 __attribute__((ext_vector_type(4), aligned(1)));

// less than 16 bytes, in one access of each size that they hold; src NULL: zeros
__device__ __forceinline__ void copy_few(char* dst, const char* src, uint32_t n) {
  typedef uint64_t u64_at_1 __attribute__((aligned(1)));
  uint32_t at = 0;
  if (n & 8) *reinterpret_cast<u64_at_1*>(dst) = src ? *reinterpret_cast<const u64_at_1*>(src) : 0, at = 8;
  if (n & 4) *reinterpret_cast<u32_at_1*>(dst + at) = src ? *reinterpret_cast<const u32_at_1*>(src + at) : 0, at += 4;
  if (n & 2) *reinterpret_cast<u16_at_1*>(dst + at) = src ? *reinterpret_cast<const u16_at_1*>(src + at) : 0, at += 2;
  if (n & 1) dst[at] = src ? src[at] : 0;
}

__global__ __launch_bounds__(AGPU_BLOCK) void take_rows_kernel(States states, uint64_t n_src, const uint32_t* idx, const uint32_t* lengths, uint32_t* flags) {
  const State& s = states.s[blockIdx.y];
  const uint32_t v0 = blockIdx.x * (AGPU_BLOCK * ROWS_UNROLL) + threadIdx.x;
  u32x4_at_1 w[ROWS_UNROLL];
  uint64_t to[ROWS_UNROLL];
  uint32_t row[ROWS_UNROLL], from[ROWS_UNROLL], held[ROWS_UNROLL];
  // what the addresses depend on first: a wait for it behind a row's load would be one for the row
#pragma unroll
  for (int u = 0; u < ROWS_UNROLL; u++) {
    const uint32_t v = v0 + u * AGPU_BLOCK, at = v < s.n_vecs ? v : 0;
    row[u] = at / s.by_row;
    from[u] = idx[row[u]];
    held[u] = lengths ? lengths[row[u]] : 0;
  }
#pragma unroll
  for (int u = 0; u < ROWS_UNROLL; u++) {
    const uint32_t v = v0 + u * AGPU_BLOCK;
    to[u] = ROW_NONE;
    w[u] = u32x4_at_1{0, 0, 0, 0};
    if (v >= s.n_vecs || from[u] == AGPU_NO_ROW) continue;
    const uint32_t in_row = v - row[u] * s.vecs_per_row, piece = in_row / s.by_piece;
    uint32_t off = (in_row - piece * s.by_piece.d) * 16, end = s.piece_bytes;
    if (lengths) {
      const uint64_t most = held[u] * s.position_bytes;
      end = most < end ? (uint32_t)most : end;
    }
    if (off >= end) continue;
    if (from[u] >= n_src) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
    const uint64_t source = from[u] * s.src_row_stride + piece * s.src_piece_stride, target = row[u] * s.dst_row_stride + piece * s.dst_piece_stride;
    if (end < 16) {
      copy_few(s.dst + target, from[u] < n_src ? s.src + source : nullptr, end);
      continue;
    }
    if (off + 16 > end) off = end - 16;
    to[u] = target + off;
    if (from[u] < n_src) w[u] = *reinterpret_cast<const u32x4_at_1*>(s.src + source + off);
  }
#pragma unroll
  for (int u = 0; u < ROWS_UNROLL; u++)
    if (to[u] != ROW_NONE) __builtin_nontemporal_store(w[u], reinterpret_cast<u32x4_at_1*>(s.dst + to[u]));
}

agpu_status check_states(int32_t n_states, const agpu_state* states, uint64_t n_src, const uint32_t* idx, const uint32_t* lengths, uint64_t n) {
  Places places[2 * 64 + 2];
  uint32_t count = 0;
  for (const uint32_t* column : {idx, lengths})
    if (column) places[count++] = {reinterpret_cast<uintptr_t>(column), 1, 0, 1, 0, 4 * n, false, -1};
  for (int32_t k = 0; k < n_states; k++) {
    const agpu_state& s = states[k];
    if (s.n_pieces == 0 || s.piece_bytes == 0) continue;
    AGPU_REQUIRE(s.dst && (s.src || n_src == 0), AGPU_ERR_ARG, "null pointer");
    uint64_t row_bytes, from, to;
    AGPU_REQUIRE(!__builtin_mul_overflow(s.n_pieces, s.piece_bytes, &row_bytes) && extent(n_src, s.src_row_stride, s.n_pieces, s.src_piece_stride, s.piece_bytes, &from) &&
                     extent(n, s.dst_row_stride, s.n_pieces, s.dst_piece_stride, s.piece_bytes, &to),
                 AGPU_ERR_SHAPE, "a state past the address space");
    AGPU_REQUIRE(disjoint(n, s.dst_row_stride, s.n_pieces, s.dst_piece_stride, s.piece_bytes), AGPU_ERR_SHAPE, "rows that are written may not overlap");
    AGPU_REQUIRE(row_bytes < (1ull << 31), AGPU_ERR_SHAPE, "a row holds less than 2^31 bytes");
    // (a length times position_bytes then stays below 2^63)
    AGPU_REQUIRE(!lengths || (s.position_bytes > 0 && s.position_bytes <= s.piece_bytes), AGPU_ERR_SHAPE, "lengths need position_bytes, at most piece_bytes");
    // (its src and its dst are compared too: rows are not reordered in place)
    places[count++] = {reinterpret_cast<uintptr_t>(s.dst), n, s.dst_row_stride, s.n_pieces, s.dst_piece_stride, s.piece_bytes, true, 2 * k};
    if (from) places[count++] = {reinterpret_cast<uintptr_t>(s.src), n_src, s.src_row_stride, s.n_pieces, s.src_piece_stride, s.piece_bytes, false, 2 * k + 1};
  }
  uint32_t x, y;
  if (overlapping(places, count, &x, &y)) {
    AGPU_REQUIRE(places[x].owner >= 0 && places[y].owner >= 0, AGPU_ERR_ARG, "a dst overlaps the indexes or the lengths");
    AGPU_REQUIRE(places[x].written && places[y].written, AGPU_ERR_ARG, "a dst overlaps a src");
    AGPU_REQUIRE(false, AGPU_ERR_ARG, "two dsts overlap");
  }
  return AGPU_OK;
}

}  // namespace

extern "C" {

agpu_status agpu_put_quantised(agpu_pipeline* p, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const uint32_t* slots, uint64_t n) {
  return quantised_slots(p, true, n_cols, stores, rows, slots, n, __func__);
}
agpu_status agpu_take_quantised(agpu_pipeline* p, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const uint32_t* slots, uint64_t n) {
  return quantised_slots(p, false, n_cols, stores, rows, slots, n, __func__);
}
agpu_status agpu_put_quantised_pages(agpu_pipeline* p, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const agpu_page_map* pages, uint64_t n) {
  return quantised_pages(p, true, n_cols, stores, rows, pages, n, __func__);
}
agpu_status agpu_take_quantised_pages(agpu_pipeline* p, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const agpu_page_map* pages, uint64_t n) {
  return quantised_pages(p, false, n_cols, stores, rows, pages, n, __func__);
}

agpu_status agpu_take_rows(agpu_pipeline* p, int32_t n_states, const agpu_state* states, uint64_t n_src, const uint32_t* idx, const uint32_t* lengths, uint64_t n) {
  AGPU_REQUIRE(n_states >= 0 && n_states <= 64, AGPU_ERR_ARG, "0 <= n_states <= 64");
  const bool any = n_states > 0 && n > 0;
  AGPU_REQUIRE(!any || (states && idx), AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(aligned_to(idx, 4) && aligned_to(lengths, 4), AGPU_ERR_SHAPE, "alignment");
  AGPU_REQUIRE(n <= (1ull << 32) && n_src <= (1ull << 32), AGPU_ERR_SHAPE, "at most 2^32 rows");
  if (any) {
    const agpu_status st = check_states(n_states, states, n_src, idx, lengths, n);
    if (st != AGPU_OK) return st;
  }
  AGPU_BIND(p);
  if (!any) return AGPU_OK;
  const auto accesses = [](const agpu_state& s) { return s.n_pieces * ((s.piece_bytes + 15) / 16); };  // of a row
  uint64_t longest = 0;
  for (int32_t k = 0; k < n_states; k++)
    if (accesses(states[k]) > longest) longest = accesses(states[k]);
  if (longest == 0) return AGPU_OK;
  // accesses are counted in 31 bits: as many rows at a time as that holds
  const uint64_t at_once = ((1ull << 31) - 1) / longest;
  for (uint64_t r0 = 0; r0 < n; r0 += at_once) {
    const uint64_t rows = n - r0 < at_once ? n - r0 : at_once;
    for (int32_t k = 0; k < n_states;) {
      States held;
      uint32_t m = 0, most = 0;
      for (; k < n_states && m < MAX_STATES; k++) {
        const agpu_state& s = states[k];
        if (s.n_pieces == 0 || s.piece_bytes == 0) continue;
        const uint32_t per_row = (uint32_t)accesses(s), per_piece = per_row / (uint32_t)s.n_pieces, n_vecs = (uint32_t)rows * per_row;
        held.s[m++] = {static_cast<const char*>(s.src), static_cast<char*>(s.dst) + r0 * s.dst_row_stride, s.src_row_stride, s.src_piece_stride, s.dst_row_stride,
                       s.dst_piece_stride, s.position_bytes, n_vecs, per_row, (uint32_t)s.piece_bytes, divide_by(per_row), divide_by(per_piece)};
        most = n_vecs > most ? n_vecs : most;
      }
      if (m == 0) break;
      const dim3 grid((most + AGPU_BLOCK * ROWS_UNROLL - 1) / (AGPU_BLOCK * ROWS_UNROLL), m);
      const uint32_t* at = idx + r0;
      const uint32_t* len = lengths ? lengths + r0 : nullptr;
      hipLaunchKernelGGL(take_rows_kernel, grid, dim3(AGPU_BLOCK), 0, p->stream, held, n_src, at, len, p->flags);
      AGPU_LAUNCH_CHECK();
    }
  }
  return AGPU_OK;
}

}  // extern "C"
