// beams.hip — beam search's selection: log-softmax over every row's vocabulary and the k best of a request's rows x tokens.
//
// One pass over the logits.  A row is cut into segments of one WAVE each; the wave streams its segment, adding up exp(x) and keeping the tokens that
// can be among its k best, and leaves (sum, k best) in the workspace.  A block a request joins the sums and selects among the segments' bests.
// No wave needs the maximum first: exp is taken relative to that of the first tile whose maximum is an ordinary number, and f32 holds it as long as
// the segment's maximum is at most 60 above that; a segment of another kind is read again.
//
// 256 rows x 128256 bf16, 8 beams, k 16 (least and average of 100 launches): segments 22.0 and 23.3 us (66 MB: 3.0 and 2.8 TB/s), join 5.8 and 6.3.  The
// segments execute 19 vector instructions a logit, 13.5 us of every SIMD — about 12 in the stream, of which the term's exp are 6 and the pair sums, the clamp, the
// unpacking and the maxima 3.5; the floors and the hits' exact terms are the rest — and the loads alone take 12.6 us; one generation of waves in step
// overlaps the two in part only.  One request (4 x 32000): 5.8 and 6.5 + 4.6 and 5.1 us, launches and latency.
//
// Precision.  The result is whole numbers, and rows that compete differ by their log-sums only: a log-sum 1e-7 off swaps tokens of two beams.  Scores are
// compared in f64.  Of the sum, the terms of the tokens that reach the floor — at least the 16 largest of a row, the bulk where it is sharp — are taken in
// f64 and left out of the f32 ones.  An f32 term is 2^f · 2^n with x log2 e = n + f, |f| <= 1/2: one fma rounds x log2 e to n, the next gives f, a third adds x
// times what log2 e has beyond f32 (2^-26 of error each), the instruction for 2^f is within 2^-23; 16 are added with 4 roundings, the rest in f64.
// That bounds a log-sum's error by 2^-23 + ln 2 · 2^-25 + 4 · 2^-24 < 3.8e-7; many different terms are off at random, and it is about 1e-9.
// What does not count (a masked logit, −infinity, one that a f64 term stands for) is e^-80 of the reference in the f32 sum: at most 8192 of them beside a
// segment's largest term, which is the reference's or larger: 8192 e^-80 < 2e-31, nothing in a f64 sum — a lone token's is exactly 1.  A tile before
// the reference's has no terms: its logits lie more than 60 below the maximum (8192 e^-60 < 8e-23), or the segment is read again.
#include "common.hpp"
#include "row_address.hpp"

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
// a segment's part of its row: sum = Σ exp(x − ref), ref its maximum; NaN where it holds a NaN or +infinity, 0 where nothing is above −infinity
struct SegSum {
  double sum, ref;
};
struct Entry {  // logit −infinity: none
  float logit;
  uint32_t token;
};

__device__ __forceinline__ bool is_finished(const BeamArgs& a, uint32_t row) { return a.finished && (a.finished[row >> 6] >> (row & 63) & 1); }

// ---------------------------------------------------------------- exp
constexpr float LOG2E = 0x1.715476p+0f, LOG2E_LOW = 0x1.4ae0cp-26f, MAGIC = 0x1.8p23f;
constexpr double LN2 = 0.69314718055994530942;
constexpr float REF_MOST = 16384.0f;  // of a reference: MAGIC − k holds its steps
constexpr float APART = 60.0f;        // of a segment's maximum above its reference; above a tile that has no terms, at least
constexpr float LEAST = 80.0f;        // of a term below the reference
// exp(x) / 2^N, k = MAGIC − N; x log2 e − N within 2^±126
__device__ __forceinline__ float exp_term(float x, float k) {
  const float z = __builtin_fmaf(x, LOG2E, k);  // its low bits: n − N
  const float f = __builtin_fmaf(x, LOG2E_LOW, __builtin_fmaf(x, LOG2E, k - z));
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, __builtin_amdgcn_exp2f(f)) + (__builtin_bit_cast(uint32_t, z) << 23));
}

// ---------------------------------------------------------------- order
constexpr float LOWEST = -__builtin_inff();
// u32 that grows with the value; −0 counts as +0
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// the k-th largest of the wave's x[0] … x[N − 1] (−infinity if there are fewer above it), found bit by bit, by how many reach the prefix.  Orders have
// `low` bits that are the same in all values of one sign: clear, of negative values set
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
  if (!(t >> 31)) t |= (1u << low) - 1;
  return t > order_of(LOWEST) ? value_of(t) : LOWEST;
}

__device__ __forceinline__ uint32_t lanes_below(uint64_t who) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0)); }

// ---------------------------------------------------------------- a segment
template <typename T> struct Raw;  // low: bits of an order that are equal in all values of the type of one sign
typedef uint32_t u32x4_at_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_at_2 __attribute__((ext_vector_type(4), aligned(2)));
template <> struct Raw<float> {
  typedef u32x4_at_4 Vector;  // 16 bytes from any element on
  static constexpr int low = 0;
  static __device__ __forceinline__ float at(u32x4 w, int i) {
    const uint32_t b = w[i];  // (a bit cast of w[i] itself takes element 0)
    return __builtin_bit_cast(float, b);
  }
};
template <> struct Raw<f16_t> {
  typedef u32x4_at_2 Vector;
  static constexpr int low = 13;
  static __device__ __forceinline__ float at(u32x4 w, int i) { return (float)__builtin_bit_cast(f16_t, (uint16_t)(w[i / 2] >> (i & 1) * 16)); }
};
template <> struct Raw<bf16_t> {
  typedef u32x4_at_2 Vector;
  static constexpr int low = 16;
  static __device__ __forceinline__ float at(u32x4 w, int i) { return __builtin_bit_cast(float, (i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16); }
};

constexpr int TILE = 1024;  // logits a wave takes at a time: 16 a lane, the next tile's on their way (two tiles ahead: no faster)
constexpr uint32_t MOST_TILES = 8;  // of a segment
constexpr int HITS = 2048;  // that it looks at twice; more: the segment is read again
constexpr uint32_t EXACT = 16;  // at least so many of the largest terms are taken in f64
constexpr int RANKED = 8;       // compared at a time
constexpr int LIST = 512;   // tokens it can keep; of logits in no order about 3 k + 10 reach the floor.  More: k passes over the segment

template <typename T, bool MASK>
struct Segment {
  static constexpr int VE = 16 / sizeof(T), U = TILE / 64 / VE;
  typedef typename Raw<T>::Vector Vector;
  const T* x;           // the row
  const uint8_t* bits;  // its allowed tokens
  uint32_t vocab, lane;

  // first token of vector u of tile t: counted from the row's start, wherever in memory that is — so a row's sum depends on its logits only, and equal
  // rows have equal scores (the loads may start at any element)
  __device__ __forceinline__ uint32_t token(uint32_t t, int u) const { return t * TILE + u * (64 * VE) + lane * VE; }
  // whether all of a tile are the row's (the same in all lanes)
  __device__ __forceinline__ bool whole(uint32_t t) const { return (t + 1) * TILE <= vocab; }

  // m: bit i: element i of the vector counts
  __device__ __forceinline__ void load(uint32_t t, u32x4 (&w)[U], uint32_t (&m)[U]) const {
    if (whole(t)) {
      const T* at = x + (uint64_t)t * TILE + lane * VE;
#pragma unroll
      for (int u = 0; u < U; u++) w[u] = *reinterpret_cast<const Vector*>(at + u * (64 * VE));
    } else {  // the row's end: whole vectors, and the one that it does not fill value by value, all on their way at once
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t at = token(t, u);
        m[u] = 0;
        w[u] = u32x4{0, 0, 0, 0};
        if (at + VE <= vocab) w[u] = *reinterpret_cast<const Vector*>(x + at), m[u] = (1u << VE) - 1;
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t at = token(t, u);
        if (at < vocab && at + VE > vocab) {
          T e[VE];
#pragma unroll
          for (int i = 0; i < VE; i++) e[i] = x[at + i < vocab ? at + i : vocab - 1];
          m[u] = (1u << (vocab - at)) - 1;
          w[u] = __builtin_bit_cast(u32x4, e);
        }
      }
    }
    if (MASK) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t at = token(t, u), b = at < vocab ? bits[at >> 3] >> (at & 7) : 0u;
        m[u] = whole(t) ? b : m[u] & b;
      }
    }
  }
  // the logits, −infinity for what is not allowed
  __device__ __forceinline__ void values(uint32_t t, const u32x4 (&w)[U], const uint32_t (&m)[U], float (&v)[U * VE]) const {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < VE; i++) v[u * VE + i] = Raw<T>::at(w[u], i);
    if (MASK || !whole(t)) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < VE; i++) v[u * VE + i] = (m[u] >> i & 1) ? v[u * VE + i] : LOWEST;
    }
  }
};

// the larger, without the instruction that would quiet a NaN first (of a NaN either: rows that hold one are found by themselves)
__device__ __forceinline__ float max_of(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// the largest, a NaN if there is one
__device__ __forceinline__ float maximum_of(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <typename T, bool MASK>
__global__ __launch_bounds__(AGPU_BLOCK) void beam_segment_kernel(BeamArgs a, uint32_t tiles, uint32_t row_blocks, SegSum* sums, Entry* entries) {
  typedef Segment<T, MASK> S;
  constexpr int VE = S::VE, U = S::U, EPT = U * VE;
  __shared__ uint64_t lists[AGPU_BLOCK / 64][LIST + RANKED];
  __shared__ float tops[AGPU_BLOCK / 64][2][64];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x / row_blocks, seg = (blockIdx.x - row * row_blocks) * waves + wave, id = row * a.segs + seg;
  const bool idle = seg >= a.segs || is_finished(a, row);  // (it keeps the others company at the barriers)
  uint64_t* list = lists[wave];

  S s;
  s.x = static_cast<const T*>(a.logits) + row * a.row_stride;
  s.bits = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  s.vocab = a.vocab;
  s.lane = lane;
  const uint32_t t0 = seg * tiles, row_tiles = (a.vocab + TILE - 1) / TILE, t1 = idle ? t0 : t0 + tiles < row_tiles ? t0 + tiles : row_tiles;

  float top[2] = {LOWEST, LOWEST};  // the largest of the lane's first and second eight logits of every tile
  float floor_v = LOWEST, above = -0x1.fffffep127f, ref_v = 0.0f, k = MAGIC, least = 0.0f, without = LOWEST;
  bool referred = false;
  double sum = 0.0;
  uint64_t nan = 0;
  uint32_t hits[4] = {0, 0, 0, 0};  // a bit a logit of the lane's, tile by tile: it reached the floor
  u32x4 two_w[2][U];  // the tile at hand and the next, on its way
  uint32_t two_m[2][U];
  if (t0 < t1) s.load(t0, two_w[0], two_m[0]);
#pragma unroll  // (the buffers and the bits' places are then fixed: 4 % of the time)
  for (uint32_t step = 0; step < MOST_TILES; step++) {
    if (step >= tiles) break;
    const uint32_t t = t0 + step;
    u32x4 (&w)[U] = two_w[step % 2];
    uint32_t (&m)[U] = two_m[step % 2];
    float v[EPT], vm[U];
    if (t < t1) {
      if (t + 1 < t1) s.load(t + 1, two_w[(step + 1) % 2], two_m[(step + 1) % 2]);
      s.values(t, w, m, v);
#pragma unroll
      for (int u = 0; u < U; u++) {
        vm[u] = maximum_of(v[u * VE], v[u * VE + 1], v[u * VE + 2]);
#pragma unroll
        for (int i = 3; i < VE; i += 2) vm[u] = maximum_of(vm[u], v[u * VE + i], v[u * VE + (i + 1 < VE ? i + 1 : i)]);
      }
#pragma unroll
      for (int u = 0; u < U; u += 2) nan |= __ballot(__builtin_isunordered(vm[u], vm[u + 1]));
      float tm[2] = {vm[0], vm[U / 2]};
#pragma unroll
      for (int u = 1; u < U / 2; u++) tm[0] = fmaxf(tm[0], vm[u]), tm[1] = fmaxf(tm[1], vm[U / 2 + u]);
      top[0] = fmaxf(top[0], tm[0]), top[1] = fmaxf(top[1], tm[1]);
      if (!referred) {  // the reference: the tile's maximum, at most REF_MOST of it (far above that the segment is read again)
        float f = fmaxf(tm[0], tm[1]);
        for (int d = 32; d; d >>= 1) f = fmaxf(f, __shfl_xor(f, d));
        f = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, f)));
        referred = f >= -REF_MOST;
        if (referred) {
          ref_v = fminf(f, REF_MOST);
          k = MAGIC - __builtin_rintf(ref_v * LOG2E);
          least = ref_v - LEAST;
        } else {
          without = fmaxf(without, f);
        }
      }
    }
    // The floor, after tiles 0 and 2: a value that k logits of the row reach, among the maxima of the block's waves, all of one row
    if (step == 0 || step == 2) {
      tops[wave][0][lane] = top[0], tops[wave][1][lane] = top[1];
      __syncthreads();
      float two[2] = {top[0], top[1]};  // the lane's largest two of them
      if (two[1] > two[0]) two[0] = top[1], two[1] = top[0];
      for (uint32_t o = 0; o < waves; o++) {  // (an idle wave's are −infinity)
        if (o == wave) continue;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float x = tops[o][h][lane], low = fminf(x, two[0]);
          two[0] = fmaxf(x, two[0]), two[1] = fmaxf(two[1], low);
        }
      }
      const float f = wave_kth(two, a.k > EXACT ? a.k : EXACT, Raw<T>::low);
      if (f > floor_v) floor_v = f, above = f;
      if (step == 0) __syncthreads();  // (before they are written again)
    }
    if (t >= t1) continue;
#pragma unroll
    for (int u = 0; u < U; u++)
      if (__any(vm[u] >= above)) {
        uint32_t h = 0;
#pragma unroll
        for (int i = VE - 1; i >= 0; i--) {
          float& x = v[u * VE + i];
          const bool hit = x >= above;
          h = h + h + hit;
          x = hit ? LOWEST : x;  // its term is taken in f64
        }
        // Very many at the floor (all that a mask has set to the lowest number): of equal ones the lower tokens come first.  Tokens rise with the lanes
        // of a vector and from vector to vector, so behind k lanes with a hit only what is above the floor counts, here and from now on
        const uint64_t who = __ballot(h != 0);
        if ((uint32_t)__popcll(who) >= a.k) {
          const bool late = lanes_below(who) >= a.k;
#pragma unroll
          for (int i = 0; i < VE; i++)
            if (late && (h >> i & 1) && Raw<T>::at(w[u], i) == floor_v) h &= ~(1u << i), v[u * VE + i] = floor_v;
          above = value_of(order_of(floor_v) + 1);
        }
        hits[step / 2] |= h << (step % 2 * EPT + u * VE);
      }
    if (!referred) continue;
    // the terms (at least e^-80 of the reference, −infinity too), added in pairs of pairs: four roundings on every way
#pragma unroll
    for (int i = 0; i < EPT; i++) v[i] = exp_term(max_of(v[i], least), k);
#pragma unroll
    for (int d = 1; d < EPT; d *= 2)
#pragma unroll
      for (int i = 0; i < EPT; i += 2 * d) v[i] += v[i + d];
    sum += (double)v[0];
  }

  float most = fmaxf(top[0], top[1]);
  for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  // the logits that reached a floor, one of each lane at a time (read again: the lane's registers cannot be indexed): their terms, and into the list
  // what reaches the last floor
  if (idle) return;
  uint32_t count = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) all += (uint32_t)__builtin_popcount(hits[i]);
  for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d);
  const bool many = all > HITS, again = most > LOWEST && most < __builtin_inff() && (many || !referred || most - ref_v > APART || most - without < APART);
  u32x4 w[U];
  uint32_t m[U];
  const double ref = most;  // (a lone token's term is then exactly 1, its log-sum the logit)
  if (most > LOWEST && !again) sum *= exp((double)(MAGIC - k) * LN2 - ref);
  if (again) {  // in f64
    sum = 0.0;
    for (uint32_t t = t0; t < t1; t++) {
      float v[EPT];
      s.load(t, w, m);
      s.values(t, w, m, v);
#pragma unroll 1
      for (int i = 0; i < EPT; i++) sum += exp((double)v[i] - ref);
    }
  }
  if (many) {
    count = LIST + 1;
  } else {
    while (__any((hits[0] | hits[1] | hits[2] | hits[3]) != 0)) {
      const int word = hits[0] ? 0 : hits[1] ? 1 : hits[2] ? 2 : 3;
      const uint32_t h = word == 0 ? hits[0] : word == 1 ? hits[1] : word == 2 ? hits[2] : hits[3];
      float y = LOWEST;
      uint32_t token = 0;
      if (h) {
        const uint32_t bit = word * 32 + __builtin_ctz(h), t = t0 + bit / EPT, i = bit % EPT;
        token = t * TILE + i / VE * (64 * VE) + lane * VE + i % VE;
        y = (float)s.x[token];
        if (!again) sum += exp((double)y - ref);
      }
      const uint32_t rest = h & (h - 1);
      hits[0] = word == 0 ? rest : hits[0], hits[1] = word == 1 ? rest : hits[1], hits[2] = word == 2 ? rest : hits[2], hits[3] = word == 3 ? rest : hits[3];
      const bool keep = y >= floor_v && y > LOWEST;
      const uint64_t who = __ballot(keep);
      const uint32_t at = count + lanes_below(who);
      if (keep && at < LIST) list[at] = (uint64_t)order_of(y) << 32 | ~token;
      count += (uint32_t)__popcll(who);
    }
  }
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (nan || most == __builtin_inff()) sum = __builtin_nan("");
  if (lane == 0) sums[id] = {most > LOWEST || sum != sum ? sum : 0.0, ref};

  Entry* out = entries + (uint64_t)id * a.k;
  if (count <= LIST) {
    if (lane >= count && lane < a.k) out[lane] = {LOWEST, 0};
    if (lane < RANKED) list[count + lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t i = lane; i < count; i += 64) {
      const uint64_t e = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < count; j += RANKED) {  // (many reads at a time: one after the other they are all latency)
        uint64_t o[RANKED];
#pragma unroll
        for (int q = 0; q < RANKED; q++) o[q] = list[j + q];
#pragma unroll
        for (int q = 0; q < RANKED; q++) rank += o[q] > e;
      }
      if (rank < a.k) out[rank] = {value_of((uint32_t)(e >> 32)), ~(uint32_t)e};
    }
  } else {  // ascending logits: the best, then the best behind it, k times
    uint64_t before = ~0ull;
    for (uint32_t r = 0; r < a.k; r++) {
      uint64_t best = 0;
      for (uint32_t t = t0; t < t1; t++) {
        float v[EPT];
        s.load(t, w, m);
        s.values(t, w, m, v);
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
// Candidates in order: score, then the lower beam, the higher logit (`tie`: smaller is better), the lower token
struct Candidate {
  double score;
  uint64_t tie;
  uint32_t token;
};
__device__ __forceinline__ Candidate candidate_of(double score, uint32_t beam, Entry x) {
  return {score, (uint64_t)beam << 32 | ~order_of(x.logit), x.token};
}
__device__ __forceinline__ bool before_equal(const Candidate& x, const Candidate& y) { return x.tie < y.tie || (x.tie == y.tie && x.token < y.token); }
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) { return x.score > y.score || (x.score == y.score && before_equal(x, y)); }

constexpr int MERGE_BLOCK = 512, MERGE_WAVES = MERGE_BLOCK / 64, MERGE_LIST = 512, HELD = 4, PARTS = 4;
constexpr uint32_t TURN = 37;  // a thread's entries are of different ranks in their segments

// The rows' log-sums, a wave a beam; then all threads over all entries of the request, for a bound that k of them reach: the k-th of each lane's two
// largest among the threads' bests.  What reaches it goes to LDS and is ranked there by counting.
__global__ __launch_bounds__(MERGE_BLOCK) void beam_merge_kernel(BeamArgs a, Divide by_row, const SegSum* sums, const Entry* entries) {
  __shared__ double lse[1024];  // per beam: its log-sum, NaN for a row whose scores are −infinity
  __shared__ float cum[1024], bests[MERGE_BLOCK];
  __shared__ double scores[MERGE_LIST + PARTS * RANKED];
  __shared__ Candidate list[MERGE_LIST];
  __shared__ uint64_t chosen[64];
  __shared__ uint32_t count;
  const uint32_t r0 = blockIdx.x * a.beams, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), total = a.beams * by_row.d;
  const double none = -__builtin_inf();
  const Entry* mine = entries + (uint64_t)r0 * by_row.d;  // (a finished row's are what an earlier call left: its log-sum, NaN, keeps them out)
  const auto place = [](uint32_t j) { return j * MERGE_BLOCK + (threadIdx.x + j * TURN) % MERGE_BLOCK; };
  if (threadIdx.x == 0) count = 0;
  Entry held[HELD];  // the thread's first
#pragma unroll
  for (uint32_t j = 0; j < HELD; j++) held[j] = place(j) < total ? mine[place(j)] : Entry{LOWEST, 0};

  for (uint32_t b = wave; b < a.beams; b += MERGE_WAVES) {
    const uint32_t row = r0 + b;
    const SegSum* parts = sums + (uint64_t)row * a.segs;
    const SegSum first = lane < a.segs ? parts[lane] : SegSum{0.0, none};
    const float c = a.scores ? a.scores[row] : 0.0f;
    const bool done = is_finished(a, row);
    double top = first.sum != 0.0 ? first.ref : none;
    for (uint32_t i = lane + 64; i < a.segs; i += 64) top = fmax(top, parts[i].sum != 0.0 ? parts[i].ref : none);
    for (int d = 32; d; d >>= 1) top = fmax(top, __shfl_xor(top, d));
    double s = 0.0;
    for (uint32_t i = lane; i < a.segs; i += 64) {
      const SegSum g = i < 64 ? first : parts[i];
      if (g.sum != 0.0) s += g.sum * exp(g.ref - top);
    }
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) lse[b] = done ? __builtin_nan("") : top + log(s), cum[b] = c;
  }
  __syncthreads();

  const auto score = [&](Entry x, uint32_t b) {
    const double s = cum[b] + ((double)x.logit - lse[b]);
    return x.logit > LOWEST && s > none ? s : none;  // (NaN: none)
  };
  // all entries, and a finished beam's only candidate: f(score, beam, entry)
  const auto each = [&](uint32_t from, const auto& f) {  // from: so many of the thread's are left out
    for (uint32_t j = from; j * MERGE_BLOCK < total; j++) {
      const uint32_t i = place(j);
      if (i >= total) continue;
      const Entry x = mine[i];
      const uint32_t b = i / by_row;
      f(score(x, b), b, x);
    }
    for (uint32_t b = threadIdx.x; b < a.beams; b += MERGE_BLOCK)
      if (is_finished(a, r0 + b) && cum[b] == cum[b]) f((double)cum[b], b, Entry{0.0f, a.end_token});
  };
  float best = LOWEST;  // rounding to f32 keeps the order, but for ties
#pragma unroll
  for (uint32_t j = 0; j < HELD; j++)
    if (place(j) < total) best = fmaxf(best, (float)score(held[j], place(j) / by_row));
  each(HELD, [&](double s, uint32_t, Entry) { best = fmaxf(best, (float)s); });
  bests[threadIdx.x] = best;
  __syncthreads();
  float two[2] = {LOWEST, LOWEST};
#pragma unroll
  for (int i = 0; i < MERGE_WAVES; i++) {
    const float x = bests[i * 64 + lane], low = fminf(x, two[0]);
    two[0] = fmaxf(x, two[0]), two[1] = fmaxf(two[1], low);
  }
  float floor_v = wave_kth(two, a.k, 0);

  const auto offer = [&](double s, uint32_t b, Entry x) {
    if (s > none && (float)s >= floor_v) {
      const uint32_t at = atomicAdd(&count, 1u);
      if (at < MERGE_LIST) scores[at] = s, list[at] = candidate_of(s, b, x);
    }
  };
#pragma unroll
  for (uint32_t j = 0; j < HELD; j++)
    if (place(j) < total) offer(score(held[j], place(j) / by_row), place(j) / by_row, held[j]);
  each(HELD, offer);
  __syncthreads();
  uint32_t n = count;
  if (n > MERGE_LIST) {  // the bound is too low for the list (k is large): any that k and at most MERGE_LIST reach, found by halving
    uint32_t low = order_of(floor_v), high = order_of(-LOWEST) + 1;
    for (uint32_t mid = low + 1; n > MERGE_LIST && high - low > 1; mid = low + (high - low) / 2) {  // (first whether the bound itself is what so many hold)
      uint32_t reach = 0;
      each(0, [&](double s, uint32_t, Entry) { reach += s > none && order_of((float)s) >= mid; });
      for (int d = 32; d; d >>= 1) reach += __shfl_xor(reach, d);
      __syncthreads();
      if (threadIdx.x == 0) count = 0;
      __syncthreads();
      if (lane == 0) atomicAdd(&count, reach);
      __syncthreads();
      const uint32_t c = count;
      if (c > MERGE_LIST) low = mid;
      else if (c < a.k) high = mid;
      else n = c, floor_v = value_of(mid);
    }
    if (n <= MERGE_LIST) {
      __syncthreads();
      if (threadIdx.x == 0) count = 0;
      __syncthreads();
      each(0, offer);
      __syncthreads();
    }
  }
  const uint32_t found = n < a.k ? n : a.k;
  const auto put = [&](uint32_t rank, const Candidate& c) {
    const uint64_t o = (uint64_t)blockIdx.x * a.k + rank;
    const uint32_t beam = (uint32_t)(c.tie >> 32);
    a.out_scores[o] = (float)c.score;
    a.out_parents[o] = r0 + beam;
    a.out_tokens[o] = c.token;
    chosen[rank] = (uint64_t)beam * a.vocab + c.token;
  };
  if (n <= MERGE_LIST) {
    if (threadIdx.x < PARTS * RANKED) scores[n + threadIdx.x] = none;
    __syncthreads();
    // PARTS lanes a candidate, each counts among its share
    const uint32_t part = threadIdx.x % PARTS;
    for (uint32_t i = threadIdx.x / PARTS; i < n; i += MERGE_BLOCK / PARTS) {
      const Candidate c = list[i];
      uint32_t rank = 0, equal = 0;
      for (uint32_t j = part * RANKED; j < n; j += PARTS * RANKED) {
        double o[RANKED];
#pragma unroll
        for (int q = 0; q < RANKED; q++) o[q] = scores[j + q];
#pragma unroll
        for (int q = 0; q < RANKED; q++) rank += o[q] > c.score, equal |= (uint32_t)(o[q] == c.score) << q;
        while (equal) {  // (itself, and tokens of one logit)
          const int q = __builtin_ctz(equal);
          equal &= equal - 1;
          rank += before_equal(list[j + q], c);
        }
      }
#pragma unroll
      for (int d = 1; d < PARTS; d *= 2) rank += __shfl_xor(rank, d);
      if (part == 0 && rank < a.k) put(rank, c);
    }
  } else {  // very many scores equal in f32: the best, then the best behind it, k times
    Candidate before = {__builtin_inf(), 0, 0};
    for (uint32_t r = 0; r < a.k; r++) {
      Candidate top = {none, ~0ull, 0};
      each(0, [&](double s, uint32_t b, Entry x) {
        const Candidate c = candidate_of(s, b, x);
        if (s > none && (r == 0 || better(before, c)) && better(c, top)) top = c;
      });
      for (int d = 32; d; d >>= 1) {
        const Candidate o = {__shfl_xor(top.score, d), __shfl_xor(top.tie, d), __shfl_xor(top.token, d)};
        if (better(o, top)) top = o;
      }
      __syncthreads();
      if (lane == 0) list[wave] = top;
      __syncthreads();
      for (int w = 0; w < MERGE_WAVES; w++)
        if (better(list[w], top)) top = list[w];
      if (threadIdx.x == 0) put(r, top);
      before = top;
    }
  }
  if (found == a.k) return;
  // the rest: (row, token) in ascending order, without the chosen ones — of the first found + (k − found) < 128 pairs as many are free
  __syncthreads();
  if (wave == 0) {
    uint32_t at = found;
    for (uint32_t f = lane; at < a.k; f += 64) {
      bool taken = false;
      for (uint32_t j = 0; j < found; j++) taken |= chosen[j] == f;
      const uint64_t free = __ballot(!taken);
      const uint32_t mine = at + lanes_below(free);
      if (!taken && mine < a.k) {
        const uint64_t o = (uint64_t)blockIdx.x * a.k + mine;
        a.out_scores[o] = LOWEST;
        a.out_parents[o] = r0 + f / a.vocab;
        a.out_tokens[o] = f % a.vocab;
      }
      at += (uint32_t)__popcll(free);
    }
  }
}

// ---------------------------------------------------------------- host
// Tiles of a segment: the fewer, the more waves share the work; the more, the fewer lists there are to join.  As many as leave 4096 waves (16 a
// CU), at most 8: 256 rows x 128256 in 4 tiles a segment take 1.2 times as long as in 8 (27.5 us beside 22.9), and 1.5 times to join.  (The type does
// not enter: the workspace does not depend on it.)
uint32_t segment_tiles(uint64_t rows, uint64_t vocab) {
  uint32_t t = MOST_TILES;
  while (t > 1 && rows * ((vocab + t * TILE - 1) / (t * TILE)) < 4096) t /= 2;
  return t;
}
uint32_t segments(uint64_t rows, uint64_t vocab) {
  const uint64_t e = (uint64_t)segment_tiles(rows, vocab) * TILE;
  return (uint32_t)((vocab + e - 1) / e);
}
// a block's waves are a row's
uint32_t block_waves(uint32_t segs) { return segs < AGPU_BLOCK / 64 ? segs : AGPU_BLOCK / 64; }
uint32_t row_blocks(uint32_t segs) { return (segs + block_waves(segs) - 1) / block_waves(segs); }

bool workspace_bytes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k, uint64_t* out) {
  if (batch == 0 || beams == 0 || vocab == 0 || k == 0 || k > 64 || beams > 1024 || k > beams * vocab || batch * beams >= (1u << 24) || vocab >= (1ull << 31)) return false;
  const uint64_t segs = segments(batch * beams, vocab);
  if (beams * segs * k >= (1ull << 31)) return false;                                                                            // a request's entries
  if (batch * beams * row_blocks((uint32_t)segs) * block_waves((uint32_t)segs) >= (1ull << 26)) return false;  // the grid's threads, 2^32
  *out = batch * beams * segs * (sizeof(SegSum) + k * sizeof(Entry));
  return true;
}

template <typename T>
void launch_segments(agpu_pipeline* p, const BeamArgs& a, SegSum* sums, Entry* entries) {
  const uint32_t rows = a.batch * a.beams, tiles = segment_tiles(rows, a.vocab), blocks = row_blocks(a.segs);
  const dim3 grid(rows * blocks), block(64 * block_waves(a.segs));
  if (a.allowed) hipLaunchKernelGGL((beam_segment_kernel<T, true>), grid, block, 0, p->stream, a, tiles, blocks, sums, entries);
  else hipLaunchKernelGGL((beam_segment_kernel<T, false>), grid, block, 0, p->stream, a, tiles, blocks, sums, entries);
}

}  // namespace

extern "C" {

agpu_status agpu_select_beams_workspace(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t k, uint64_t* out_bytes) {
  AGPU_REQUIRE(out_bytes, AGPU_ERR_ARG, "null argument");
  *out_bytes = 0;
  if (batch == 0) return AGPU_OK;
  AGPU_REQUIRE(workspace_bytes(batch, beams, vocab, k, out_bytes), AGPU_ERR_SHAPE,
               "1 <= k <= 64, k <= beams * vocab, 1 <= beams <= 1024, batch * beams < 2^24, 1 <= vocab < 2^31, batch * beams * vocab < 2^38, "
               "beams * k * vocab < 2^43");
  return AGPU_OK;
}

agpu_status agpu_select_beams(agpu_pipeline* p, const agpu_beams* args) {
  AGPU_REQUIRE(args, AGPU_ERR_ARG, "null argument");
  const agpu_beams& b = *args;
  AGPU_REQUIRE(b.row_type >= AGPU_ROW_F32 && b.row_type <= AGPU_ROW_BF16, AGPU_ERR_ARG, "row type");
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
  AGPU_REQUIRE(b.allowed_stride % 8 == 0 && (b.allowed_stride == 0 || b.allowed_stride >= agpu_bitmap_bytes(b.vocab)), AGPU_ERR_SHAPE,
               "allowed_stride: 0, or a multiple of 8 that holds vocab bits");
  AGPU_REQUIRE(aligned_to(b.logits, b.row_type == AGPU_ROW_F32 ? 4 : 2) && aligned_to(b.scores, 4) && aligned_to(b.allowed, 8) && aligned_to(b.finished, 8) &&
                   aligned_to(b.out_scores, 4) && aligned_to(b.out_parents, 4) && aligned_to(b.out_tokens, 4) && aligned16(b.workspace),
               AGPU_ERR_SHAPE, "alignment");
  // a request's block writes while another's still reads: results do not go where scores and finished rows come from, nor the segments' where logits do
  const uint64_t found = 4ull * b.batch * b.k, rows = (uint64_t)b.batch * b.beams, item = b.row_type == AGPU_ROW_F32 ? 4 : 2;
  const auto apart = [](const void* x, uint64_t nx, const void* y, uint64_t ny) {
    const uintptr_t i = reinterpret_cast<uintptr_t>(x), j = reinterpret_cast<uintptr_t>(y);
    return !y || (i <= j ? nx <= j - i : ny <= i - j);
  };
  const void* outs[] = {b.out_scores, b.out_parents, b.out_tokens};
  for (int i = 0; i < 3; i++) {
    AGPU_REQUIRE(apart(outs[i], found, b.scores, 4 * rows), AGPU_ERR_ARG, "an output overlaps the scores");
    AGPU_REQUIRE(apart(outs[i], found, b.finished, agpu_bitmap_bytes(rows)), AGPU_ERR_ARG, "an output overlaps the finished rows");
    AGPU_REQUIRE(apart(outs[i], found, b.workspace, need), AGPU_ERR_ARG, "an output overlaps the workspace");
    for (int j = 0; j < i; j++) AGPU_REQUIRE(apart(outs[i], found, outs[j], found), AGPU_ERR_ARG, "two outputs overlap");
  }
  uint64_t span;
  AGPU_REQUIRE(b.row_stride < (1ull << 61) && extent(rows, item * b.row_stride, 1, 0, item * b.vocab, &span), AGPU_ERR_SHAPE, "logits past the address space");
  const uint64_t masks = (rows - 1) * b.allowed_stride + agpu_bitmap_bytes(b.vocab);
  AGPU_REQUIRE(apart(b.workspace, need, b.logits, span) && apart(b.workspace, need, b.scores, 4 * rows) && apart(b.workspace, need, b.finished, agpu_bitmap_bytes(rows)) &&
                   apart(b.workspace, need, b.allowed, masks), AGPU_ERR_ARG, "the workspace overlaps an input");
  AGPU_BIND(p);
  const BeamArgs a = {b.logits, b.row_stride, b.batch, b.beams, b.vocab, b.k, b.end_token, b.scores, static_cast<const uint8_t*>(b.allowed), b.allowed_stride,
                      static_cast<const uint64_t*>(b.finished), b.out_scores, b.out_parents, b.out_tokens, segments((uint64_t)b.batch * b.beams, b.vocab)};
  SegSum* sums = static_cast<SegSum*>(b.workspace);
  Entry* entries = reinterpret_cast<Entry*>(sums + (uint64_t)b.batch * b.beams * a.segs);
  if (b.row_type == AGPU_ROW_F32) launch_segments<float>(p, a, sums, entries);
  else if (b.row_type == AGPU_ROW_F16) launch_segments<f16_t>(p, a, sums, entries);
  else launch_segments<bf16_t>(p, a, sums, entries);
  AGPU_LAUNCH_CHECK();
  hipLaunchKernelGGL(beam_merge_kernel, dim3(b.batch), dim3(MERGE_BLOCK), 0, p->stream, a, divide_by(a.segs * a.k), sums, entries);
  AGPU_LAUNCH_CHECK();
  return AGPU_OK;
}

}  // extern "C"
