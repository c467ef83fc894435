// beams.hip — beam search's selection: log-softmax over every row's vocabulary and the k best of a request's rows x tokens.
//
// One pass over the logits.  A row is cut into segments of one WAVE each; the wave streams its segment, adding up exp(x) and keeping the tokens that
// can be among its k best, and leaves (sum, k best) in the workspace.  A block a request joins the sums and selects among the segments' bests.
// No wave waits for another before the join, and none needs the maximum first: f64 holds exp(x − first tile's maximum) for all x of a row
// whose logits are less than 600 apart; a segment that holds others is read again.
//
// Why 64 bits: the result is whole numbers, and rows that compete differ by their log-sums only — a log-sum 1e-7 off swaps tokens of two beams.
// The f64 unit runs at the rate of the f32 one here, so exp is made there: with c = ln 2 / 256, x = (256 e + j + r) c, |r| <= 1/2,
// exp(x) = 2^e · 2^(j/256) · (1 + r c + r² c² / 2), the middle factor from a table in LDS.  The cubic term that is left out is at most 4.2e-10, and
// odd: over many tokens it cancels.
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
// a segment's part of its row: sum = Σ exp(x − ref), NaN where it holds a NaN or +infinity, 0 where nothing is above −infinity
struct SegSum {
  double sum, ref;
};
struct Entry {  // logit −infinity: none
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

constexpr double EXP_C = 0.69314718055994530942 / EXP_STEPS, EXP_SCALE = EXP_STEPS / 0.69314718055994530942, EXP_MAGIC = 0x1.8p52;
// exp(x − ref), ref = (EXP_MAGIC − k) · EXP_C a whole number of steps: no subtraction, the steps of ref leave with the whole number.  |x| <= 2^30
__device__ __forceinline__ void add_exp(double& sum, double x, double k, const double* table) {
  const double z = __builtin_fma(x, EXP_SCALE, k);  // its low word: steps of x, less those of ref
  const int n = (int)__builtin_bit_cast(uint64_t, z);
  const double r = __builtin_fma(x, EXP_SCALE, k - z), f = __builtin_ldexp(table[n & (EXP_STEPS - 1)], n >> 8);
  sum = __builtin_fma(f, __builtin_fma(r, __builtin_fma(r, EXP_C * EXP_C / 2, EXP_C), 1.0), sum);
}

// ---------------------------------------------------------------- order
constexpr float LOWEST = -__builtin_inff();
// u32 that grows with the value; −0 counts as +0
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// a value that at least k of the wave's 64 (x[0], … x[N − 1] of every lane) reach, −infinity if there are none: the k-th largest, its bits below
// `low` cleared — found bit by bit, by how many reach the prefix
template <int N>
__device__ __forceinline__ float wave_kth(const float (&x)[N], uint32_t k, int low) {
  uint32_t o[N], t = 0;
#pragma unroll
  for (int i = 0; i < N; i++) o[i] = order_of(x[i]);
  for (int b = 31; b >= low; b--) {
    const uint32_t up = t | 1u << b;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += (uint32_t)__popcll(__ballot(o[i] >= up));
    t = n >= k ? up : t;
  }
  return t > order_of(LOWEST) ? value_of(t) : LOWEST;
}

// ---------------------------------------------------------------- a segment
template <typename T> struct Raw;  // low: bits of an order that are equal in all values of the type of one sign
template <> struct Raw<float> {
  static constexpr int low = 0;
  static __device__ __forceinline__ float at(u32x4 w, int i) {
    const uint32_t b = w[i];  // (a bit cast of w[i] itself takes element 0)
    return __builtin_bit_cast(float, b);
  }
};
template <> struct Raw<f16_t> {
  static constexpr int low = 13;
  static __device__ __forceinline__ float at(u32x4 w, int i) { return (float)__builtin_bit_cast(f16_t, (uint16_t)(w[i / 2] >> (i & 1) * 16)); }
};
template <> struct Raw<bf16_t> {
  static constexpr int low = 16;
  static __device__ __forceinline__ float at(u32x4 w, int i) { return __builtin_bit_cast(float, (i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16); }
};

constexpr int TILE = 1024;  // logits a wave takes at a time: 16 a lane
constexpr int LIST = 512;   // tokens it can keep: 18 + 9 + 6 + … for k = 16 and logits in no order, 230 for k = 64

template <typename T, bool MASK>
struct Segment {
  static constexpr int VE = 16 / sizeof(T), U = TILE / 64 / VE;
  const T* x;           // the row
  const uint8_t* bits;  // its allowed tokens
  uint32_t vocab, lead, lane;

  // first token of vector u of tile t: vectors lie on 16 bytes, the row starts `lead` elements into its first
  __device__ __forceinline__ int64_t token(uint32_t t, int u) const { return (int64_t)t * TILE + u * (64 * VE) + lane * VE - lead; }

  __device__ __forceinline__ void load(uint32_t t, u32x4 (&w)[U], uint32_t (&m)[U]) const {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t at = token(t, u);
      if (at >= 0 && at + VE <= vocab) {
        w[u] = *reinterpret_cast<const u32x4*>(x + at);
        m[u] = ~0u;
      } else {  // the row's ends
        T e[VE] = {};
        m[u] = 0;
#pragma unroll
        for (int i = 0; i < VE; i++)
          if (at + i >= 0 && at + i < vocab) e[i] = x[at + i], m[u] |= 1u << i;
        w[u] = __builtin_bit_cast(u32x4, e);
      }
      if (MASK && m[u]) {
        const uint32_t first = at < 0 ? 0u : (uint32_t)at, byte = first >> 3, last = (vocab - 1) >> 3;
        const uint32_t b = (bits[byte] | (uint32_t)bits[byte < last ? byte + 1 : last] << 8) >> (first & 7);
        m[u] &= at < 0 ? b << -at : b;
      }
    }
  }
  // the logits, −infinity for what is not allowed
  __device__ __forceinline__ void values(const u32x4 (&w)[U], const uint32_t (&m)[U], float (&v)[U * VE]) const {
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int i = 0; i < VE; i++) v[u * VE + i] = Raw<T>::at(w[u], i);
      if (MASK || !__all(m[u] == ~0u)) {
#pragma unroll
        for (int i = 0; i < VE; i++) v[u * VE + i] = (m[u] >> i & 1) ? v[u * VE + i] : LOWEST;
      }
    }
  }
};

template <typename T, bool MASK>
__global__ __launch_bounds__(AGPU_BLOCK) void beam_segment_kernel(BeamArgs a, uint32_t tiles, uint32_t n_segs, SegSum* sums, Entry* entries) {
  typedef Segment<T, MASK> S;
  constexpr int VE = S::VE, U = S::U, EPT = U * VE;
  __shared__ double table[EXP_STEPS];
  __shared__ uint64_t lists[AGPU_BLOCK / 64][LIST];
  table[threadIdx.x] = exp_table.v[threadIdx.x];
  __syncthreads();  // the only one: from here on every wave is by itself
  const uint32_t id = __builtin_amdgcn_readfirstlane(blockIdx.x * (AGPU_BLOCK / 64) + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
  if (id >= n_segs) return;
  const uint32_t row = id / a.segs, seg = id - row * a.segs;
  if (is_finished(a, row)) return;
  uint64_t* list = lists[threadIdx.x >> 6];

  S s;
  s.x = static_cast<const T*>(a.logits) + row * a.row_stride;
  s.bits = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  s.vocab = a.vocab;
  s.lead = (uint32_t)(reinterpret_cast<uintptr_t>(s.x) & 15) / sizeof(T);
  s.lane = lane;
  const uint32_t t0 = seg * tiles, row_tiles = (uint32_t)(((uint64_t)a.vocab + s.lead + TILE - 1) / TILE), t1 = t0 + tiles < row_tiles ? t0 + tiles : row_tiles;

  float top[2] = {LOWEST, LOWEST};  // the largest of the lane's first and second eight logits of every tile
  float floor_v = LOWEST, ref_v = 0.0f;
  double sum = 0.0, k = EXP_MAGIC;
  uint32_t count = 0, negative_nan = 0;
  u32x4 w[U], next[U];
  uint32_t m[U], next_m[U];
  if (t0 < t1) s.load(t0, w, m);
  for (uint32_t t = t0; t < t1; t++) {
    if (t + 1 < t1) s.load(t + 1, next, next_m);
    float v[EPT];
    s.values(w, m, v);
    float tm[2] = {v[0], v[EPT / 2]};
#pragma unroll
    for (int i = 1; i < EPT / 2; i++) tm[0] = fmaxf(tm[0], v[i]), tm[1] = fmaxf(tm[1], v[EPT / 2 + i]);
    top[0] = fmaxf(top[0], tm[0]), top[1] = fmaxf(top[1], tm[1]);
    if (t == t0) {  // the reference: the tile's maximum, as far as it is an ordinary number
      float f = fmaxf(tm[0], tm[1]);
      for (int d = 32; d; d >>= 1) f = fmaxf(f, __shfl_xor(f, d));
      ref_v = __builtin_fabsf(f) <= 16384.0f ? f : 0.0f;
      k = EXP_MAGIC - __builtin_rint((double)ref_v * EXP_SCALE);
    }
    if (__any(fmaxf(tm[0], tm[1]) >= floor_v)) {
      if (((t - t0) & (t - t0 + 1)) == 0) floor_v = wave_kth(top, a.k, Raw<T>::low);  // tiles 0, 1, 3, 7 …
      const float above = fmaxf(floor_v, -0x1.fffffep127f);
#pragma unroll
      for (int i = 0; i < EPT; i++) {
        const uint64_t who = __ballot(v[i] >= above);
        if (who) {
          const uint32_t at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
          if (v[i] >= above && at < LIST) list[at] = (uint64_t)order_of(v[i]) << 32 | ~(uint32_t)(s.token(t, i / VE) + i % VE);
          count += (uint32_t)__popcll(who);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < EPT; i++) {
      // at least −2^30: the unsigned order of negative numbers grows downwards.  It keeps +infinity and positive NaN, which make the sum NaN
      const uint32_t b = __builtin_bit_cast(uint32_t, v[i]), low = 0xCE800000u;
      negative_nan = b > negative_nan ? b : negative_nan;
      add_exp(sum, (double)__builtin_bit_cast(float, b < low ? b : low), k, table);
    }
#pragma unroll
    for (int u = 0; u < U; u++) w[u] = next[u], m[u] = next_m[u];
  }

  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  float most = fmaxf(top[0], top[1]);
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  double ref = (EXP_MAGIC - k) * EXP_C;
  if (most > LOWEST && most < __builtin_inff() && __builtin_fabsf(most - ref_v) > 600.0f) {  // again, below the maximum that is now known
    ref = most;
    sum = 0.0;
    for (uint32_t t = t0; t < t1; t++) {
      float v[EPT];
      s.load(t, w, m);
      s.values(w, m, v);
#pragma unroll
      for (int i = 0; i < EPT; i++) {
        const double d = (double)v[i] - ref;
        add_exp(sum, d < -0x1p30 ? -0x1p30 : d, EXP_MAGIC, table);
      }
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  }
  if (__any(negative_nan > 0xFF800000u) || most == __builtin_inff()) sum = __builtin_nan("");
  if (lane == 0) sums[id] = {most > LOWEST || sum != sum ? sum : 0.0, ref};

  Entry* out = entries + (uint64_t)id * a.k;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the list was written by other lanes
  if (count <= LIST) {
    if (lane >= count && lane < a.k) out[lane] = {LOWEST, 0};
    for (uint32_t i = lane; i < count; i += 64) {
      const uint64_t e = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < count; j++) rank += list[j] > e;
      if (rank < a.k) out[rank] = {value_of((uint32_t)(e >> 32)), ~(uint32_t)e};
    }
  } else {  // very many equal logits, or ascending ones: the best, then the best behind it, k times
    uint64_t before = ~0ull;
    for (uint32_t r = 0; r < a.k; r++) {
      uint64_t best = 0;
      for (uint32_t t = t0; t < t1; t++) {
        float v[EPT];
        s.load(t, w, m);
        s.values(w, m, v);
#pragma unroll
        for (int i = 0; i < EPT; i++) {
          const uint64_t e = (uint64_t)order_of(v[i]) << 32 | ~(uint32_t)(s.token(t, i / VE) + i % VE);
          if (e < before && e > best && v[i] > LOWEST) best = e;
        }
      }
      for (int d = 32; d; d >>= 1) {
        const uint64_t o = __shfl_xor(best, d);
        best = o > best ? o : best;
      }
      if (lane == 0) out[r] = {value_of((uint32_t)(best >> 32)), ~(uint32_t)best};
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

constexpr int MERGE_BLOCK = 1024, MERGE_LIST = 512, HELD = 4;

// Lists of k entries, best first: the largest scores among a few heads of them give a bound that k candidates reach; what reaches it goes to LDS and
// is ranked there by counting.
__global__ __launch_bounds__(MERGE_BLOCK) void beam_merge_kernel(BeamArgs a, const SegSum* sums, const Entry* entries) {
  __shared__ double lse[1024];  // per beam: its log-sum, NaN for a row whose scores are −infinity
  __shared__ float cum[1024];
  __shared__ Candidate list[MERGE_LIST];
  __shared__ uint64_t chosen[64];
  __shared__ uint32_t count;
  const uint32_t r0 = blockIdx.x * a.beams, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per_row = a.segs * a.k, n = a.beams * per_row;
  const double none = -__builtin_inf();
  entries += (uint64_t)r0 * per_row;
  Entry held[HELD], heads[HELD];
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    const uint32_t e = threadIdx.x + i * MERGE_BLOCK;
    held[i] = e < n ? entries[e] : Entry{LOWEST, 0};
  }
  // a sample of the lists' heads, one wave's: `deep` of each
  const uint32_t lists = a.beams * a.segs, deep = lists < a.k ? (a.k + lists - 1) / lists : 1;
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    const uint32_t h = lane + i * 64;
    heads[i] = h < lists * deep ? entries[h / deep * a.k + h % deep] : Entry{LOWEST, 0};
  }
  if (threadIdx.x == 0) count = 0;
  for (uint32_t b = wave; b < a.beams; b += MERGE_BLOCK / 64) {
    const bool done = is_finished(a, r0 + b);
    double s = 0.0, ref = none;
    if (!done)
      for (uint32_t i = lane; i < a.segs; i += 64) {
        const SegSum g = sums[(uint64_t)(r0 + b) * a.segs + i];
        if (g.sum == 0.0) continue;
        if (g.ref > ref) s = s * exp(ref - g.ref) + g.sum, ref = g.ref;
        else s += g.sum * exp(g.ref - ref);
      }
    double top = ref;
    for (int d = 32; d; d >>= 1) top = fmax(top, __shfl_xor(top, d));
    s = ref > none ? s * exp(ref - top) : 0.0;
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) lse[b] = done ? __builtin_nan("") : top + log(s), cum[b] = a.scores ? a.scores[r0 + b] : 0.0f;
  }
  __syncthreads();

  const auto candidate = [&](uint32_t e, Entry x) {
    const uint32_t b = e / per_row;
    Candidate c = {none, b, x.token, x.logit};
    const double s = (double)cum[b] + ((double)x.logit - lse[b]);
    if (x.logit > LOWEST && s > none) c.score = s;  // (NaN: none)
    return c;
  };
  float best[1] = {LOWEST};  // rounding to f32 keeps the order, but for ties
#pragma unroll
  for (int i = 0; i < HELD; i++) {
    const uint32_t h = lane + i * 64;
    if (h < lists * deep) best[0] = fmaxf(best[0], (float)candidate(h / deep * a.k, heads[i]).score);
  }
  for (uint32_t h = lane + HELD * 64; h < lists * deep; h += 64) {
    const uint32_t e = h / deep * a.k + h % deep;
    best[0] = fmaxf(best[0], (float)candidate(e, entries[e]).score);
  }
  const float floor_v = wave_kth(best, a.k, 0);
  const auto offer = [&](const Candidate& c) {
    if (c.score > none && (float)c.score >= floor_v) {
      const uint32_t at = atomicAdd(&count, 1u);
      if (at < MERGE_LIST) list[at] = c;
    }
  };
#pragma unroll
  for (int i = 0; i < HELD; i++)
    if (threadIdx.x + i * MERGE_BLOCK < n) offer(candidate(threadIdx.x + i * MERGE_BLOCK, held[i]));
  for (uint32_t e = threadIdx.x + HELD * MERGE_BLOCK; e < n; e += MERGE_BLOCK) offer(candidate(e, entries[e]));
  // a finished row's one candidate (of its entries none was: its log-sum is NaN)
  for (uint32_t b = threadIdx.x; b < a.beams; b += MERGE_BLOCK)
    if (is_finished(a, r0 + b)) offer({cum[b] == cum[b] ? (double)cum[b] : none, b, a.end_token, 0.0f});
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
    for (uint32_t i = threadIdx.x; i < count; i += MERGE_BLOCK) {
      const Candidate c = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < count; j++) rank += better(list[j], c);
      if (rank < a.k) put(rank, c);
    }
  } else {  // very many equal scores: the best, then the best behind it, k times
    Candidate before = {__builtin_inf(), 0, 0, 0.0f};
    for (uint32_t r = 0; r < a.k; r++) {
      Candidate top = {none, ~0u, 0, 0.0f};
      const auto take = [&](const Candidate& c) {
        if (c.score > none && (r == 0 || better(before, c)) && better(c, top)) top = c;
      };
      for (uint32_t e = threadIdx.x; e < n; e += MERGE_BLOCK) take(candidate(e, entries[e]));
      for (uint32_t b = threadIdx.x; b < a.beams; b += MERGE_BLOCK)
        if (is_finished(a, r0 + b)) take({cum[b] == cum[b] ? (double)cum[b] : none, b, a.end_token, 0.0f});
      for (int d = 32; d; d >>= 1) {
        const Candidate o = {__shfl_xor(top.score, d), __shfl_xor(top.beam, d), __shfl_xor(top.token, d), __shfl_xor(top.logit, d)};
        if (better(o, top)) top = o;
      }
      __syncthreads();
      if (lane == 0) list[wave] = top;
      __syncthreads();
      for (int w = 0; w < MERGE_BLOCK / 64; w++)
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
// Tiles of a segment: the fewer, the more waves share the work; the more, the fewer lists there are to join.  As many as leave 4096 waves (16 a
// CU), at most 8.  (The type does not enter: the workspace does not depend on it.)
uint32_t segment_tiles(uint64_t rows, uint64_t vocab) {
  uint32_t t = 8;
  while (t > 1 && rows * ((vocab + 7 + t * TILE - 1) / (t * TILE)) < 4096) t /= 2;
  return t;
}
uint32_t segments(uint64_t rows, uint64_t vocab) {
  const uint64_t e = (uint64_t)segment_tiles(rows, vocab) * TILE;
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
  const uint32_t rows = a.batch * a.beams, n = rows * a.segs, tiles = segment_tiles(rows, a.vocab);
  const dim3 grid((n + AGPU_BLOCK / 64 - 1) / (AGPU_BLOCK / 64));
  if (a.allowed) hipLaunchKernelGGL((beam_segment_kernel<T, true>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, tiles, n, sums, entries);
  else hipLaunchKernelGGL((beam_segment_kernel<T, false>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, tiles, n, sums, entries);
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
  hipLaunchKernelGGL(beam_merge_kernel, dim3(b.batch), dim3(MERGE_BLOCK), 0, p->stream, a, sums, entries);
  AGPU_LAUNCH_CHECK();
  return AGPU_OK;
}

}  // extern "C"
