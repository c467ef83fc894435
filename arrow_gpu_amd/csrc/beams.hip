// beams.hip — beam search's selection: log-softmax over every row's vocabulary and the k best of a request's rows x tokens.
//
// One pass over the logits.  A row is cut into segments of one block each, whose logits stay in registers: the segment's maximum M, the sum of
// exp(x − M), and its k best tokens go to the workspace; a block a request joins the segments (log-sum-exp as M + log S, sums rescaled by
// exp(M' − M)) and selects among the segments' bests by score.
//
// Why 64 bits: the result is whole numbers, and rows that compete differ by their log-sums only — a log-sum 1e-7 off swaps tokens of two beams.
// The f64 unit runs at the rate of the f32 one here, so exp is made there: x − M = (256 e + j + r) · c, c = ln 2 / 256, |r| <= 1/2, exp = 2^e · 2^(j/256) ·
// (1 + r c + r² c² / 2), the middle factor from a table in LDS.  The cubic term that is left out is at most 4.2e-10 and odd: over many tokens it
// cancels.
#include "common.hpp"

namespace {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

struct BeamArgs {
  const void* logits;
  uint64_t row_stride;
  uint32_t batch, beams, vocab, k, end_token;
  const float* scores;
  const uint8_t* allowed;
  uint64_t allowed_stride;
  const uint64_t* finished;
  float* out_scores;
  uint32_t* out_parents;
  uint32_t* out_tokens;
  uint32_t segs;
};
// a segment's part of its row; count: how many of its k entries there are, BAD: it holds a NaN or +infinity
struct SegSum {
  double sum;
  float max;
  uint32_t count;
};
constexpr uint32_t BAD = 0xFFFFFFFFu;
struct Entry {
  float logit;
  uint32_t token;
};

__device__ __forceinline__ bool is_finished(const BeamArgs& a, uint32_t row) { return a.finished && (a.finished[row >> 6] >> (row & 63) & 1); }

// ---------------------------------------------------------------- exp
constexpr int EXP_STEPS = 256;
struct ExpTable {
  double v[EXP_STEPS];
};
constexpr ExpTable make_exp_table() {
  ExpTable t = {};
  for (int j = 0; j < EXP_STEPS; j++) {  // Taylor's series of exp(j ln 2 / 256), arguments below 0.7: 20 terms
    const double y = 0.69314718055994530942 * j / EXP_STEPS;
    double term = 1.0, sum = 0.0;
    for (int n = 1; n <= 20; n++) sum += term, term = term * y / n;
    t.v[j] = sum;
  }
  return t;
}
__device__ const ExpTable exp_table = make_exp_table();

// exp(d), d = x − M <= 0
__device__ __forceinline__ double exp_of(double d, const double* table) {
  const double magic = 0x1.8p52, scale = EXP_STEPS / 0.69314718055994530942, c = 0.69314718055994530942 / EXP_STEPS;
  d = fmax(d, -690.0);  // 1e-300, nothing beside the maximum's 1; −infinity too
  const double z = __builtin_fma(d, scale, magic);  // its low word: the whole number nearest to d · 256 / ln 2
  const int n = (int)__builtin_bit_cast(uint64_t, z);
  const double r = __builtin_fma(d, scale, magic - z), f = table[n & (EXP_STEPS - 1)];
  const double p = __builtin_fma(r, __builtin_fma(r, c * c / 2, c), 1.0);
  return __builtin_ldexp(p * f, n >> 8);
}

// ---------------------------------------------------------------- order
// u32 that grows with the value; −0 counts as +0
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// the k-th largest of a wave's values: bit by bit, how many lanes reach the prefix.  `low`: bits that are 0 in every value, or do not matter
__device__ __forceinline__ uint32_t wave_kth(uint32_t v, uint32_t k, int low) {
  uint32_t t = 0;
  for (int b = 31; b >= low; b--)
    if ((uint32_t)__popcll(__ballot(v >= (t | 1u << b))) >= k) t |= 1u << b;
  return t;
}

// ---------------------------------------------------------------- a segment
template <typename T> struct Raw;  // what an order's low bits hold
template <> struct Raw<float> { static constexpr int low = 0; };
template <> struct Raw<f16_t> { static constexpr int low = 13; };  // (of negative values these bits are all set: the prefix lies below, and still above the next)
template <> struct Raw<bf16_t> { static constexpr int low = 16; };

constexpr int LIST = 512;

template <typename T, int VPT>
__global__ __launch_bounds__(AGPU_BLOCK) void beam_segment_kernel(BeamArgs a, SegSum* sums, Entry* entries) {
  constexpr int VE = 16 / sizeof(T), EPT = VPT * VE;
  __shared__ double table[EXP_STEPS];
  __shared__ double wave_sum[AGPU_BLOCK / 64];
  __shared__ uint64_t list[LIST];
  __shared__ float wave_max[AGPU_BLOCK / 64];
  __shared__ uint32_t wave_t[AGPU_BLOCK / 64], wave_bad[AGPU_BLOCK / 64], count;
  const uint32_t row = blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs, wave = threadIdx.x >> 6;
  if (is_finished(a, row)) return;
  table[threadIdx.x] = exp_table.v[threadIdx.x];
  if (threadIdx.x == 0) count = 0;

  // vectors on 16 bytes; the row starts `lead` elements into the first
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T);
  const uint8_t* bits = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  const uint32_t last_byte = (a.vocab - 1) >> 3;
  float v[EPT];
  bool bad = false;
  float tm = -__builtin_inff();
#pragma unroll
  for (int u = 0; u < VPT; u++) {
    const int64_t at = ((int64_t)seg * VPT + u) * AGPU_BLOCK * VE + threadIdx.x * VE - lead;
    if (at >= 0 && at + VE <= a.vocab) {
      typedef T vec __attribute__((ext_vector_type(VE)));
      const vec w = *reinterpret_cast<const vec*>(x + at);
#pragma unroll
      for (int i = 0; i < VE; i++) v[u * VE + i] = (float)w[i];
    } else {
#pragma unroll
      for (int i = 0; i < VE; i++) v[u * VE + i] = at + i >= 0 && at + i < a.vocab ? (float)x[at + i] : -__builtin_inff();
    }
    if (bits && at + VE > 0 && at < a.vocab) {
      const uint32_t t = at < 0 ? 0u : (uint32_t)at, byte = t >> 3;
      uint32_t m = (bits[byte] | (uint32_t)bits[byte < last_byte ? byte + 1 : byte] << 8) >> (t & 7);
      if (at < 0) m <<= -at;
#pragma unroll
      for (int i = 0; i < VE; i++) v[u * VE + i] = (m >> i & 1) ? v[u * VE + i] : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < VE; i++) {
      bad |= !(v[u * VE + i] < __builtin_inff());
      tm = fmaxf(tm, v[u * VE + i]);
    }
  }

  // the wave's maximum, and a value that at least k of its logits reach: the k-th largest of the lanes' maxima
  float m = tm;
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const uint32_t t = wave_kth(order_of(tm), a.k, Raw<T>::low);
  bad = __any(bad);
  if ((threadIdx.x & 63) == 0) wave_max[wave] = m, wave_t[wave] = t, wave_bad[wave] = bad;
  __syncthreads();
  m = wave_max[0];
  uint32_t least = wave_t[0], any_bad = wave_bad[0];
#pragma unroll
  for (int w = 1; w < AGPU_BLOCK / 64; w++) {
    m = fmaxf(m, wave_max[w]);
    least = least > wave_t[w] ? least : wave_t[w];
    any_bad |= wave_bad[w];
  }
  SegSum* mine = sums + (uint64_t)row * a.segs + seg;
  if (any_bad || m == -__builtin_inff()) {  // nothing to select here
    if (threadIdx.x == 0) *mine = {0.0, m, any_bad ? BAD : 0u};
    return;
  }

  const double top = m;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < EPT; i++) sum += exp_of((double)v[i] - top, table);
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) wave_sum[wave] = sum;

  // what reaches the block's threshold, as (logit, token) in one number: larger is better
  const float floor_v = least > order_of(-__builtin_inff()) ? value_of(least) : -__builtin_inff();
  if (order_of(tm) >= least && tm > -__builtin_inff()) {
#pragma unroll
    for (int u = 0; u < VPT; u++)
#pragma unroll
      for (int i = 0; i < VE; i++)
        if (v[u * VE + i] >= floor_v && v[u * VE + i] > -__builtin_inff()) {
          const uint32_t at = atomicAdd(&count, 1u);
          if (at < LIST) list[at] = (uint64_t)order_of(v[u * VE + i]) << 32 | ~(((seg * VPT + u) * AGPU_BLOCK + threadIdx.x) * VE + i - lead);
        }
  }
  __syncthreads();
  const uint32_t n = count;
  Entry* out = entries + ((uint64_t)row * a.segs + seg) * a.k;
  if (threadIdx.x == 0) *mine = {wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3], m, n < a.k ? n : a.k};
  if (n <= LIST) {
    for (uint32_t i = threadIdx.x; i < n; i += AGPU_BLOCK) {
      const uint64_t e = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; j++) rank += list[j] > e;
      if (rank < a.k) out[rank] = {value_of((uint32_t)(e >> 32)), ~(uint32_t)e};
    }
  } else {  // very many equal logits: the best, then the best behind it, k times
    uint64_t before = ~0ull;
    for (uint32_t r = 0; r < a.k; r++) {
      uint64_t best = 0;
#pragma unroll
      for (int u = 0; u < VPT; u++)
#pragma unroll
        for (int i = 0; i < VE; i++) {
          const uint64_t e = (uint64_t)order_of(v[u * VE + i]) << 32 | ~(((seg * VPT + u) * AGPU_BLOCK + threadIdx.x) * VE + i - lead);
          if (e < before && e > best && v[u * VE + i] > -__builtin_inff()) best = e;
        }
      for (int d = 32; d; d >>= 1) {
        const uint64_t o = __shfl_xor(best, d);
        best = o > best ? o : best;
      }
      __syncthreads();
      if ((threadIdx.x & 63) == 0) list[wave] = best;
      __syncthreads();
      for (int w = 0; w < AGPU_BLOCK / 64; w++) best = list[w] > best ? list[w] : best;
      if (threadIdx.x == 0) out[r] = {value_of((uint32_t)(best >> 32)), ~(uint32_t)best};
      before = best;
    }
  }
}

// ---------------------------------------------------------------- a request
struct Candidate {
  double score;
  uint32_t beam, token;
  float logit;
};
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) {
  if (x.score != y.score) return x.score > y.score;
  if (x.beam != y.beam) return x.beam < y.beam;
  if (x.logit != y.logit) return x.logit > y.logit;
  return x.token < y.token;
}

constexpr int MERGE_LIST = 512;

__global__ __launch_bounds__(AGPU_BLOCK) void beam_merge_kernel(BeamArgs a, const SegSum* sums, const Entry* entries) {
  __shared__ double lse[1024];  // per beam: its log-sum, NaN for a row whose scores are −infinity
  __shared__ Candidate list[MERGE_LIST];
  __shared__ uint64_t chosen[64];
  __shared__ uint32_t wave_t[AGPU_BLOCK / 64], count;
  const uint32_t r0 = blockIdx.x * a.beams, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per_row = a.segs * a.k, n = a.beams * per_row;
  const double none = -__builtin_inf();
  if (threadIdx.x == 0) count = 0;
  for (uint32_t b = wave; b < a.beams; b += AGPU_BLOCK / 64) {
    double m = none, s = 0.0;
    bool bad = false;
    if (!is_finished(a, r0 + b))
      for (uint32_t i = lane; i < a.segs; i += 64) {
        const SegSum g = sums[(uint64_t)(r0 + b) * a.segs + i];
        bad |= g.count == BAD;
        if (g.max > m) s = s * exp(m - (double)g.max) + g.sum, m = g.max;
        else if (g.max > -__builtin_inff()) s += g.sum * exp((double)g.max - m);
      }
    double top = m;
    for (int d = 32; d; d >>= 1) top = fmax(top, __shfl_xor(top, d));
    if (m > none) s *= exp(m - top);
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) lse[b] = top + log(s);  // (nothing allowed: NaN or −infinity, and no entries)
    if (__any(bad) && lane == 0) lse[b] = __builtin_nan("");
  }
  __syncthreads();

  // entry e → its candidate; score −infinity: none
  const auto candidate = [&](uint32_t e) {
    const uint32_t b = e / per_row, i = e - b * per_row, row = r0 + b;
    Candidate c = {none, b, 0, 0.0f};
    const double cum = a.scores ? (double)a.scores[row] : 0.0;
    double s = none;
    if (is_finished(a, row)) {
      if (i == 0) s = cum, c.token = a.end_token;
    } else {
      const uint32_t seg = i / a.k, held = sums[(uint64_t)row * a.segs + seg].count;
      if (held != BAD && i - seg * a.k < held) {
        const Entry x = entries[(uint64_t)row * per_row + i];
        s = cum + ((double)x.logit - lse[b]);
        c.token = x.token, c.logit = x.logit;
      }
    }
    if (s > none) c.score = s;  // (NaN: none)
    return c;
  };

  float best = -__builtin_inff();  // rounding to f32 keeps the order, but for ties
  for (uint32_t e = threadIdx.x; e < n; e += AGPU_BLOCK) best = fmaxf(best, (float)candidate(e).score);
  const uint32_t t = wave_kth(order_of(best), a.k, 0);
  if (lane == 0) wave_t[wave] = t;
  __syncthreads();
  uint32_t least = wave_t[0];
  for (int w = 1; w < AGPU_BLOCK / 64; w++) least = least > wave_t[w] ? least : wave_t[w];
  const float floor_v = value_of(least);
  for (uint32_t e = threadIdx.x; e < n; e += AGPU_BLOCK) {
    const Candidate c = candidate(e);
    if (c.score > none && (float)c.score >= floor_v) {
      const uint32_t at = atomicAdd(&count, 1u);
      if (at < MERGE_LIST) list[at] = c;
    }
  }
  __syncthreads();
  const uint32_t found = count < a.k ? count : a.k;
  const auto put = [&](uint32_t rank, const Candidate& c) {
    const uint64_t o = (uint64_t)blockIdx.x * a.k + rank;
    a.out_scores[o] = (float)c.score;
    a.out_parents[o] = r0 + c.beam;
    a.out_tokens[o] = c.token;
    chosen[rank] = (uint64_t)c.beam * a.vocab + c.token;
  };
  if (count <= MERGE_LIST) {
    for (uint32_t i = threadIdx.x; i < count; i += AGPU_BLOCK) {
      const Candidate c = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < count; j++) rank += better(list[j], c);
      if (rank < a.k) put(rank, c);
    }
  } else {  // very many equal scores: the best, then the best behind it, k times
    Candidate before = {__builtin_inf(), 0, 0, 0.0f};
    for (uint32_t r = 0; r < a.k; r++) {
      Candidate top = {none, ~0u, 0, 0.0f};
      for (uint32_t e = threadIdx.x; e < n; e += AGPU_BLOCK) {
        const Candidate c = candidate(e);
        if (c.score > none && (r == 0 || better(before, c)) && better(c, top)) top = c;
      }
      for (int d = 32; d; d >>= 1) {
        const Candidate o = {__shfl_xor(top.score, d), __shfl_xor(top.beam, d), __shfl_xor(top.token, d), __shfl_xor(top.logit, d)};
        if (better(o, top)) top = o;
      }
      __syncthreads();
      if (lane == 0) list[wave] = top;
      __syncthreads();
      for (int w = 0; w < AGPU_BLOCK / 64; w++)
        if (better(list[w], top)) top = list[w];
      if (threadIdx.x == 0) put(r, top);
      before = top;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0)  // the rest: (row, token) in ascending order, without the chosen ones
    for (uint64_t f = 0, i = found; i < a.k; f++) {
      bool taken = false;
      for (uint32_t j = 0; j < found; j++) taken |= chosen[j] == f;
      if (taken) continue;
      const uint64_t o = (uint64_t)blockIdx.x * a.k + i++;
      a.out_scores[o] = -__builtin_inff();
      a.out_parents[o] = r0 + (uint32_t)(f / a.vocab);
      a.out_tokens[o] = (uint32_t)(f % a.vocab);
    }
}

// ---------------------------------------------------------------- host
// Segments of a row: the type does not enter, so that the workspace does not depend on it
constexpr uint32_t SEG_MOST = 8192, SEG_LEAST = 2048;
uint32_t segment_elements(uint64_t rows, uint64_t vocab) {
  uint32_t e = SEG_MOST;
  while (e > SEG_LEAST && rows * ((vocab + 7 + e - 1) / e) < 512) e /= 2;
  return e;
}
uint32_t segments(uint64_t rows, uint64_t vocab) {
  const uint32_t e = segment_elements(rows, vocab);
  return (uint32_t)((vocab + 7 + e - 1) / e);  // + 7: a row may start anywhere in a vector
}

bool workspace_bytes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k, uint64_t* out) {
  if (batch == 0 || beams == 0 || vocab == 0 || k == 0 || k > 64 || beams > 1024 || k > beams * vocab || batch * beams >= (1u << 24) || vocab >= (1ull << 31)) return false;
  const uint64_t segs = segments(batch * beams, vocab);
  if (beams * segs * k >= (1ull << 32) || batch * beams * segs >= (1ull << 31)) return false;  // a request's entries, the blocks
  *out = batch * beams * segs * (sizeof(SegSum) + k * sizeof(Entry));
  return true;
}

template <typename T>
void launch_segments(agpu_pipeline* p, const BeamArgs& a, SegSum* sums, Entry* entries) {
  constexpr int E = 16 / sizeof(T) * AGPU_BLOCK;
  const dim3 grid(a.batch * a.beams * a.segs);
  switch (segment_elements((uint64_t)a.batch * a.beams, a.vocab)) {
    case SEG_MOST: hipLaunchKernelGGL((beam_segment_kernel<T, SEG_MOST / E>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, sums, entries); break;
    case SEG_MOST / 2: hipLaunchKernelGGL((beam_segment_kernel<T, SEG_MOST / 2 / E>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, sums, entries); break;
    default: hipLaunchKernelGGL((beam_segment_kernel<T, SEG_LEAST / E>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, sums, entries); break;
  }
}

}  // namespace

extern "C" {

agpu_status agpu_select_beams_workspace(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t k, uint64_t* out_bytes) {
  AGPU_REQUIRE(out_bytes, AGPU_ERR_ARG, "null argument");
  *out_bytes = 0;
  if (batch == 0) return AGPU_OK;
  AGPU_REQUIRE(workspace_bytes(batch, beams, vocab, k, out_bytes), AGPU_ERR_SHAPE,
               "1 <= k <= 64, k <= beams * vocab, 1 <= beams <= 1024, batch * beams < 2^24, 1 <= vocab < 2^31");
  return AGPU_OK;
}

agpu_status agpu_select_beams(agpu_pipeline* p, const agpu_beams* args) {
  AGPU_REQUIRE(args, AGPU_ERR_ARG, "null argument");
  const agpu_beams& b = *args;
  AGPU_REQUIRE(b.type >= AGPU_ROW_F32 && b.type <= AGPU_ROW_BF16, AGPU_ERR_ARG, "row type");
  if (b.batch == 0) {
    AGPU_BIND(p);
    return AGPU_OK;
  }
  uint64_t need = 0;
  const agpu_status st = agpu_select_beams_workspace(b.batch, b.beams, b.vocab, b.k, &need);
  if (st != AGPU_OK) return st;
  AGPU_REQUIRE(b.logits && b.out_scores && b.out_parents && b.out_tokens && b.workspace, AGPU_ERR_ARG, "null pointer");
  AGPU_REQUIRE(b.workspace_bytes >= need, AGPU_ERR_SHAPE, "workspace too small");
  AGPU_REQUIRE(b.end_token < b.vocab, AGPU_ERR_SHAPE, "end_token < vocab");
  AGPU_REQUIRE(b.batch * b.beams == 1 || b.row_stride >= b.vocab, AGPU_ERR_SHAPE, "row_stride >= vocab");
  AGPU_REQUIRE(b.allowed_stride % 8 == 0 && (b.allowed_stride == 0 || b.allowed_stride >= agpu_bitmap_bytes(b.vocab)), AGPU_ERR_SHAPE,
               "allowed_stride: 0, or a multiple of 8 that holds vocab bits");
  AGPU_REQUIRE(aligned_to(b.logits, b.type == AGPU_ROW_F32 ? 4 : 2) && aligned_to(b.scores, 4) && aligned_to(b.allowed, 8) && aligned_to(b.finished, 8) &&
                   aligned_to(b.out_scores, 4) && aligned_to(b.out_parents, 4) && aligned_to(b.out_tokens, 4) && aligned16(b.workspace),
               AGPU_ERR_SHAPE, "alignment");
  AGPU_BIND(p);
  const BeamArgs a = {b.logits, b.row_stride, b.batch, b.beams, b.vocab, b.k, b.end_token, b.scores, static_cast<const uint8_t*>(b.allowed), b.allowed_stride,
                      static_cast<const uint64_t*>(b.finished), b.out_scores, b.out_parents, b.out_tokens, segments((uint64_t)b.batch * b.beams, b.vocab)};
  SegSum* sums = static_cast<SegSum*>(b.workspace);
  Entry* entries = reinterpret_cast<Entry*>(sums + (uint64_t)b.batch * b.beams * a.segs);
  if (b.type == AGPU_ROW_F32) launch_segments<float>(p, a, sums, entries);
  else if (b.type == AGPU_ROW_F16) launch_segments<f16_t>(p, a, sums, entries);
  else launch_segments<bf16_t>(p, a, sums, entries);
  AGPU_LAUNCH_CHECK();
  hipLaunchKernelGGL(beam_merge_kernel, dim3(b.batch), dim3(AGPU_BLOCK), 0, p->stream, a, sums, entries);
  AGPU_LAUNCH_CHECK();
  return AGPU_OK;
}

}  // extern "C"
