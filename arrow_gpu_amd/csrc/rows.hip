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
// span: max |x| or max − min; bad: the group holds a NaN or an infinity
template <int CODE>
__device__ __forceinline__ Factors factors(float span, float lo, bool bad) {
  const float top = Top<CODE>::v;
  if (bad || !(span < __builtin_inff())) return {__builtin_nanf(""), 0.0f, lo};
  if (span < top * 0x1p-126f) return {0.0f, 0.0f, lo};  // span / top would be subnormal and top / span could overflow
  return {span / top, top / span, lo};
}
__device__ __forceinline__ uint32_t whole(float x, float inv) {  // low byte: the code in two's complement
  return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, inv, 0x1.8p23f));
}

// ---------------------------------------------------------------- one wave a group: any group, stride and alignment
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

template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void put_group_kernel(QuantCol c, QuantShape q, RowAddr addr, uint64_t n_groups, uint32_t* flags) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t waves = (uint64_t)gridDim.x * (AGPU_BLOCK / 64);
  for (uint64_t g = (uint64_t)blockIdx.x * (AGPU_BLOCK / 64) + (threadIdx.x >> 6); g < n_groups; g += waves) {
    const uint64_t row = g / q.groups_per_row;
    const uint32_t in_row = (uint32_t)(g - row * q.groups_per_row), head = in_row / q.groups_per_head;
    const uint64_t slot = row_slot(addr, row, c.n_slots);
    if (slot >= ROW_BAD) {
      if (slot == ROW_BAD && lane == 0) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
      continue;
    }
    const T* x = static_cast<const T*>(c.x) + row * c.row_stride + head * c.head_stride + (in_row - head * q.groups_per_head) * q.group;
    float lo = __builtin_inff(), hi = -__builtin_inff();
    bool bad = false;
    for (uint32_t i = lane; i < q.group; i += 64) {
      const float v = (float)x[i];
      bad |= !(__builtin_fabsf(v) < __builtin_inff());
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
    }
    for (int s = 32; s; s >>= 1) {
      lo = fminf(lo, __shfl_xor(lo, s));
      hi = fmaxf(hi, __shfl_xor(hi, s));
    }
    bad = __any(bad);
    const Factors f = factors<CODE>(CODE == AGPU_CODE_I4 ? hi - lo : fmaxf(hi, -lo), lo, bad);
    const uint64_t at = slot * q.groups_per_row + in_row;
    if (CODE == AGPU_CODE_I4) {
      if (lane == 0) c.scales[2 * at] = f.scale, c.scales[2 * at + 1] = f.lo;
      for (uint32_t i = lane; i < q.group / 2; i += 64)
        c.codes[at * (q.group / 2) + i] = (uint8_t)((whole((float)x[2 * i] - f.lo, f.inv) & 15) | (whole((float)x[2 * i + 1] - f.lo, f.inv) & 15) << 4);
    } else {
      if (lane == 0) c.scales[at] = f.scale;
      for (uint32_t i = lane; i < q.group; i += 64) {
        const float v = (float)x[i];
        c.codes[at * q.group + i] = CODE == AGPU_CODE_I8 ? (uint8_t)whole(v, f.inv)
                                                         : (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v * f.inv, 0.0f, 0, false);
      }
    }
  }
}

template <typename T, int CODE>
__global__ __launch_bounds__(AGPU_BLOCK) void take_group_kernel(QuantCol c, QuantShape q, RowAddr addr, uint64_t n_groups, uint32_t* flags) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t waves = (uint64_t)gridDim.x * (AGPU_BLOCK / 64);
  for (uint64_t g = (uint64_t)blockIdx.x * (AGPU_BLOCK / 64) + (threadIdx.x >> 6); g < n_groups; g += waves) {
    const uint64_t row = g / q.groups_per_row;
    const uint32_t in_row = (uint32_t)(g - row * q.groups_per_row), head = in_row / q.groups_per_head;
    const uint64_t slot = row_slot(addr, row, c.n_slots);
    if (slot == ROW_NONE) continue;
    const bool ok = slot != ROW_BAD;
    if (!ok && lane == 0) *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
    T* x = static_cast<T*>(c.x) + row * c.row_stride + head * c.head_stride + (in_row - head * q.groups_per_head) * q.group;
    const uint64_t at = slot * q.groups_per_row + in_row;
    const float scale = !ok ? 0.0f : c.scales[CODE == AGPU_CODE_I4 ? 2 * at : at], lo = ok && CODE == AGPU_CODE_I4 ? c.scales[2 * at + 1] : 0.0f;
    for (uint32_t i = lane; i < q.group; i += 64) {
      float v = 0.0f;
      if (ok && CODE == AGPU_CODE_I4) v = __builtin_fmaf((float)((c.codes[(at * q.group + i) / 2] >> (4 * (i & 1))) & 15), scale, lo);
      else if (ok && CODE == AGPU_CODE_I8) v = (float)(int8_t)c.codes[at * q.group + i] * scale;
      else if (ok) v = __builtin_amdgcn_cvt_f32_fp8(c.codes[at * q.group + i], 0) * scale;
      x[i] = (T)v;
    }
  }
}

// ---------------------------------------------------------------- host: checks and dispatch
agpu_status check_columns(int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, uint64_t n, bool writes_rows) {
  for (int32_t k = 0; k < n_cols; k++) {
    const agpu_quantised_rows& s = stores[k];
    const agpu_rows& r = rows[k];
    AGPU_REQUIRE(r.type >= AGPU_ROW_F32 && r.type <= AGPU_ROW_BF16, AGPU_ERR_ARG, "row type");
    AGPU_REQUIRE(s.code >= AGPU_CODE_I8 && s.code <= AGPU_CODE_E4M3, AGPU_ERR_ARG, "code type");
    AGPU_REQUIRE(s.heads > 0 && s.dim > 0 && (uint64_t)s.heads * s.dim <= (1u << 30), AGPU_ERR_SHAPE, "1 <= heads * dim <= 2^30");
    AGPU_REQUIRE(s.group > 0 && s.group <= 65536 && s.dim % s.group == 0, AGPU_ERR_SHAPE, "group divides dim, 1 <= group <= 65536");
    AGPU_REQUIRE(s.code != AGPU_CODE_I4 || s.group % 2 == 0, AGPU_ERR_SHAPE, "4-bit codes: an even group");
    AGPU_REQUIRE(s.n_slots <= (1ull << 32), AGPU_ERR_SHAPE, "n_slots <= 2^32");
    AGPU_REQUIRE(r.data && s.codes && s.scales, AGPU_ERR_ARG, "null pointer");
    AGPU_REQUIRE(aligned_to(r.data, r.type == AGPU_ROW_F32 ? 4 : 2) && aligned_to(s.scales, 4), AGPU_ERR_SHAPE, "alignment");
    if (writes_rows) {
      const uint64_t hs = s.heads > 1 ? r.head_stride : s.dim, rs = n > 1 ? r.row_stride : (uint64_t)-1;
      AGPU_REQUIRE(hs >= s.dim && rs >= s.dim, AGPU_ERR_SHAPE, "rows that are written may not overlap");
    }
  }
  return AGPU_OK;
}

template <typename T, int CODE>
agpu_status launch_groups(agpu_pipeline* p, bool put, const QuantCol& c, const QuantShape& q, const RowAddr& addr, uint64_t n) {
  const uint64_t n_groups = n * q.groups_per_row;
  const uint64_t blocks = (n_groups + 3) / 4;
  const int grid = (int)(blocks > (1u << 20) ? (1u << 20) : blocks);
  if (put) hipLaunchKernelGGL((put_group_kernel<T, CODE>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, c, q, addr, n_groups, p->flags);
  else hipLaunchKernelGGL((take_group_kernel<T, CODE>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, c, q, addr, n_groups, p->flags);
  AGPU_LAUNCH_CHECK();
  return AGPU_OK;
}
template <typename T>
agpu_status launch_code(agpu_pipeline* p, bool put, int code, const QuantCol& c, const QuantShape& q, const RowAddr& addr, uint64_t n) {
  switch (code) {
    case AGPU_CODE_I8: return launch_groups<T, AGPU_CODE_I8>(p, put, c, q, addr, n);
    case AGPU_CODE_I4: return launch_groups<T, AGPU_CODE_I4>(p, put, c, q, addr, n);
    default: return launch_groups<T, AGPU_CODE_E4M3>(p, put, c, q, addr, n);
  }
}

agpu_status quantised(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const RowAddr& addr,
                      uint64_t n, const char* name) {
  AGPU_BIND_AS(p, name);
  if (n == 0) return AGPU_OK;
  for (int32_t k = 0; k < n_cols; k++) {
    const agpu_quantised_rows& s = stores[k];
    const agpu_rows& r = rows[k];
    const QuantCol c = {r.data, r.row_stride, r.head_stride, static_cast<uint8_t*>(s.codes), s.scales, s.n_slots};
    const QuantShape q = {s.heads, s.dim, s.group, s.dim / s.group, s.heads * (s.dim / s.group)};
    const agpu_status st = r.type == AGPU_ROW_F32   ? launch_code<float>(p, put, s.code, c, q, addr, n)
                           : r.type == AGPU_ROW_F16 ? launch_code<f16_t>(p, put, s.code, c, q, addr, n)
                                                    : launch_code<bf16_t>(p, put, s.code, c, q, addr, n);
    if (st != AGPU_OK) return st;
  }
  return AGPU_OK;
}

agpu_status quantised_slots(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const uint32_t* slots,
                            uint64_t n, const char* name) {
  AGPU_REQUIRE(n_cols >= 0 && n_cols <= 64, AGPU_ERR_ARG, "0 <= n_cols <= 64");
  RowAddr a = {};
  if (n_cols == 0 || n == 0) return quantised(p, put, 0, stores, rows, a, 0, name);
  AGPU_REQUIRE(stores && rows && slots, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(n <= (1ull << 32), AGPU_ERR_SHAPE, "n <= 2^32");
  AGPU_REQUIRE(aligned_to(slots, 4), AGPU_ERR_SHAPE, "alignment");
  const agpu_status st = check_columns(n_cols, stores, rows, n, !put);
  if (st != AGPU_OK) return st;
  a.slots = slots;
  return quantised(p, put, n_cols, stores, rows, a, n, name);
}

agpu_status quantised_pages(agpu_pipeline* p, bool put, int32_t n_cols, const agpu_quantised_rows* stores, const agpu_rows* rows, const agpu_page_map* m,
                            uint64_t n, const char* name) {
  AGPU_REQUIRE(n_cols >= 0 && n_cols <= 64, AGPU_ERR_ARG, "0 <= n_cols <= 64");
  if (n_cols == 0 || n == 0) return quantised(p, put, 0, stores, rows, RowAddr{}, 0, name);
  AGPU_REQUIRE(stores && rows && m && m->offsets, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(n <= (1ull << 32), AGPU_ERR_SHAPE, "n <= 2^32");
  AGPU_REQUIRE(m->n_seqs > 0 && m->n_seqs < (1u << 31) && m->page_rows > 0, AGPU_ERR_SHAPE, "1 <= n_seqs < 2^31, page_rows >= 1");
  AGPU_REQUIRE(m->max_pages == 0 || m->tables, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(aligned_to(m->tables, 4) && aligned_to(m->offsets, 4) && aligned_to(m->first, 4), AGPU_ERR_SHAPE, "alignment");
  const agpu_status st = check_columns(n_cols, stores, rows, n, !put);
  if (st != AGPU_OK) return st;
  const RowAddr a = {nullptr, m->tables, m->table_stride, m->offsets, m->first, m->n_seqs, m->max_pages, m->page_rows};
  return quantised(p, put, n_cols, stores, rows, a, n, name);
}

// ---------------------------------------------------------------- take_rows
template <typename V>
__global__ __launch_bounds__(AGPU_BLOCK) void take_rows_kernel(agpu_state s, uint64_t n_src, const uint32_t* idx, const uint32_t* lengths, uint64_t n_vecs,
                                                               uint64_t vecs_per_piece, uint32_t* flags) {
  const uint64_t stride = (uint64_t)gridDim.x * AGPU_BLOCK, vecs_per_row = vecs_per_piece * s.n_pieces;
  for (uint64_t v = (uint64_t)blockIdx.x * AGPU_BLOCK + threadIdx.x; v < n_vecs; v += stride) {
    const uint64_t row = v / vecs_per_row, in_row = v - row * vecs_per_row, piece = in_row / vecs_per_piece, off = (in_row - piece * vecs_per_piece) * sizeof(V);
    if (lengths && off >= lengths[row] * s.position_bytes) continue;
    const uint32_t from = idx[row];
    if (from == AGPU_NO_ROW) continue;
    V w = {};
    if (from < n_src) w = *reinterpret_cast<const V*>(static_cast<const char*>(s.src) + from * s.src_row_stride + piece * s.src_piece_stride + off);
    else *reinterpret_cast<volatile uint32_t*>(flags) = AGPU_FLAG_INDEX_RANGE;
    *reinterpret_cast<V*>(static_cast<char*>(s.dst) + row * s.dst_row_stride + piece * s.dst_piece_stride + off) = w;
  }
}

// bytes from the first to behind the last of n rows; 0: none.  false: past 2^63
bool extent(uint64_t n, uint64_t row_stride, uint64_t pieces, uint64_t piece_stride, uint64_t piece_bytes, uint64_t* out) {
  uint64_t a, b;
  if (n == 0 || pieces == 0 || piece_bytes == 0) {
    *out = 0;
    return true;
  }
  return !__builtin_mul_overflow(n - 1, row_stride, &a) && !__builtin_mul_overflow(pieces - 1, piece_stride, &b) && !__builtin_add_overflow(a, b, &a) &&
         !__builtin_add_overflow(a, piece_bytes, out) && *out < (1ull << 63);
}

agpu_status check_states(int32_t n_states, const agpu_state* states, uint64_t n_src, const uint32_t* lengths, uint64_t n) {
  for (int32_t k = 0; k < n_states; k++) {
    const agpu_state& s = states[k];
    if (s.n_pieces == 0 || s.piece_bytes == 0) continue;
    AGPU_REQUIRE(s.dst && (s.src || n_src == 0), AGPU_ERR_ARG, "null pointer");
    uint64_t row_bytes, from, to;
    AGPU_REQUIRE(!__builtin_mul_overflow(s.n_pieces, s.piece_bytes, &row_bytes) && extent(n_src, s.src_row_stride, s.n_pieces, s.src_piece_stride, s.piece_bytes, &from) &&
                     extent(n, s.dst_row_stride, s.n_pieces, s.dst_piece_stride, s.piece_bytes, &to),
                 AGPU_ERR_SHAPE, "a state past the address space");
    AGPU_REQUIRE((s.n_pieces == 1 || s.dst_piece_stride >= s.piece_bytes) && (n == 1 || s.dst_row_stride >= s.piece_bytes), AGPU_ERR_SHAPE,
                 "rows that are written may not overlap");
    AGPU_REQUIRE(!lengths || s.position_bytes > 0, AGPU_ERR_SHAPE, "lengths need position_bytes");
    for (int32_t j = 0; j < n_states; j++) {
      const agpu_state& o = states[j];
      uint64_t there;
      if (!extent(n_src, o.src_row_stride, o.n_pieces, o.src_piece_stride, o.piece_bytes, &there) || there == 0) continue;
      const uintptr_t d = reinterpret_cast<uintptr_t>(s.dst), f = reinterpret_cast<uintptr_t>(o.src);
      AGPU_REQUIRE(d + to <= f || f + there <= d, AGPU_ERR_ARG, "a dst overlaps a src");
    }
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
    const agpu_status st = check_states(n_states, states, n_src, lengths, n);
    if (st != AGPU_OK) return st;
  }
  AGPU_BIND(p);
  if (!any) return AGPU_OK;
  for (int32_t k = 0; k < n_states; k++) {
    const agpu_state& s = states[k];
    if (s.n_pieces == 0 || s.piece_bytes == 0) continue;
    // the widest access that everything is a multiple of
    const uint64_t all = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | s.src_row_stride | s.src_piece_stride | s.dst_row_stride |
                         s.dst_piece_stride | s.piece_bytes | (lengths ? s.position_bytes : 0);
    const uint64_t width = (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : 1;
    const uint64_t vecs_per_piece = s.piece_bytes / width, n_vecs = n * s.n_pieces * vecs_per_piece;
    const uint64_t blocks = (n_vecs + AGPU_BLOCK - 1) / AGPU_BLOCK;
    const int grid = (int)(blocks > (1u << 20) ? (1u << 20) : blocks);
    if (width == 16) hipLaunchKernelGGL((take_rows_kernel<u32x4>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, s, n_src, idx, lengths, n_vecs, vecs_per_piece, p->flags);
    else if (width == 4) hipLaunchKernelGGL((take_rows_kernel<uint32_t>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, s, n_src, idx, lengths, n_vecs, vecs_per_piece, p->flags);
    else hipLaunchKernelGGL((take_rows_kernel<uint8_t>), dim3(grid), dim3(AGPU_BLOCK), 0, p->stream, s, n_src, idx, lengths, n_vecs, vecs_per_piece, p->flags);
    AGPU_LAUNCH_CHECK();
  }
  return AGPU_OK;
}

}  // extern "C"
