// beams.hip — beam search's selection: log-softmax over every row's vocabulary and the k best of a request's rows x tokens.
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
};
// one row's best tokens: `count` live ones (score above −infinity), by logit, then token
struct RowBest {
  double lse;
  uint32_t count, void_row;
};
struct Entry {
  float logit;
  uint32_t token;
};

__device__ __forceinline__ bool is_allowed(const BeamArgs& a, uint32_t row, uint32_t v) {
  return !a.allowed || (a.allowed[row * a.allowed_stride + (v >> 3)] >> (v & 7) & 1);
}
__device__ __forceinline__ bool is_finished(const BeamArgs& a, uint32_t row) { return a.finished && (a.finished[row >> 6] >> (row & 63) & 1); }

// the best of a wave's, then a block's candidates (better: larger first, then smaller at); every thread gets it
__device__ __forceinline__ void block_best(double& s, uint64_t& at, double* ls, uint64_t* la) {
  for (int d = 32; d; d >>= 1) {
    const double os = __shfl_xor(s, d);
    const uint64_t oa = __shfl_xor(at, d);
    if (os > s || (os == s && oa < at)) s = os, at = oa;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) ls[threadIdx.x >> 6] = s, la[threadIdx.x >> 6] = at;
  __syncthreads();
  s = ls[0], at = la[0];
  for (int w = 1; w < AGPU_BLOCK / 64; w++)
    if (ls[w] > s || (ls[w] == s && la[w] < at)) s = ls[w], at = la[w];
}

template <typename T>
__global__ __launch_bounds__(AGPU_BLOCK) void beam_rows_kernel(BeamArgs a, RowBest* rows, Entry* entries) {
  __shared__ double ls[AGPU_BLOCK / 64];
  __shared__ uint64_t la[AGPU_BLOCK / 64];
  const uint32_t row = blockIdx.x;
  if (is_finished(a, row)) return;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  double m = -__builtin_inf();
  uint64_t none = 0;
  uint32_t bad = 0;
  for (uint32_t v = threadIdx.x; v < a.vocab; v += AGPU_BLOCK)
    if (is_allowed(a, row, v)) {
      const float f = (float)x[v];
      bad |= !(f < __builtin_inff());
      m = fmax(m, (double)f);
    }
  block_best(m, none, ls, la);
  const bool void_row = __syncthreads_or(bad) || !(m > -__builtin_inf());
  double sum = 0;
  if (!void_row)
    for (uint32_t v = threadIdx.x; v < a.vocab; v += AGPU_BLOCK)
      if (is_allowed(a, row, v)) sum += exp((double)x[v] - m);
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) ls[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double lse = m + log(ls[0] + ls[1] + ls[2] + ls[3]);
  uint32_t count = 0;
  double last = __builtin_inf();
  uint64_t last_at = 0;
  for (; count < a.k && !void_row; count++) {
    double best = -__builtin_inf();
    uint64_t at = ~0ull;
    for (uint32_t v = threadIdx.x; v < a.vocab; v += AGPU_BLOCK)
      if (is_allowed(a, row, v)) {
        const double f = (float)x[v];
        if ((f < last || (f == last && v > last_at)) && f > best) best = f, at = v;
      }
    block_best(best, at, ls, la);
    if (at == ~0ull) break;
    last = best, last_at = at;
    if (threadIdx.x == 0) entries[(uint64_t)row * a.k + count] = {(float)best, (uint32_t)at};
  }
  if (threadIdx.x == 0) rows[row] = {lse, count, void_row};
}

__global__ __launch_bounds__(AGPU_BLOCK) void beam_merge_kernel(BeamArgs a, const RowBest* rows, const Entry* entries) {
  __shared__ double ls[AGPU_BLOCK / 64];
  __shared__ uint64_t la[AGPU_BLOCK / 64];
  __shared__ uint64_t chosen[64];
  const uint32_t r0 = blockIdx.x * a.beams, n = a.beams * a.k;
  double last = __builtin_inf();
  uint64_t last_at = 0;
  uint32_t count = 0;
  for (; count < a.k; count++) {
    double best = -__builtin_inf();
    uint64_t at = ~0ull;
    for (uint32_t e = threadIdx.x; e < n; e += AGPU_BLOCK) {
      const uint32_t b = e / a.k, row = r0 + b, i = e - b * a.k;
      const double cum = a.scores ? a.scores[row] : 0.0f;
      double s = -__builtin_inf();
      if (is_finished(a, row)) {
        if (i == 0) s = cum;
      } else if (!rows[row].void_row && i < rows[row].count) {
        s = cum + ((double)entries[(uint64_t)row * a.k + i].logit - rows[row].lse);
      }
      if ((count == 0 || s < last || (s == last && e > last_at)) && (s > best)) best = s, at = e;
    }
    block_best(best, at, ls, la);
    if (at == ~0ull) break;
    last = best, last_at = at;
    if (threadIdx.x == 0) {
      const uint32_t row = r0 + (uint32_t)at / a.k, token = is_finished(a, row) ? a.end_token : entries[(uint64_t)row * a.k + at % a.k].token;
      const uint64_t o = (uint64_t)blockIdx.x * a.k + count;
      a.out_scores[o] = (float)best;
      a.out_parents[o] = row;
      a.out_tokens[o] = token;
      chosen[count] = (uint64_t)(row - r0) * a.vocab + token;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0)  // the rest: (row, token) in ascending order, without the chosen ones
    for (uint64_t f = 0, i = count; i < a.k; f++) {
      bool taken = false;
      for (uint32_t j = 0; j < count; j++) taken |= chosen[j] == f;
      if (taken) continue;
      const uint64_t o = (uint64_t)blockIdx.x * a.k + i++;
      a.out_scores[o] = -__builtin_inff();
      a.out_parents[o] = r0 + (uint32_t)(f / a.vocab);
      a.out_tokens[o] = (uint32_t)(f % a.vocab);
    }
}

bool workspace_bytes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k, uint64_t* out) {
  if (batch == 0 || beams == 0 || vocab == 0 || k == 0 || k > 64 || beams > 1024 || k > beams * vocab || batch * beams >= (1u << 24) || vocab >= (1ull << 31)) return false;
  *out = batch * beams * (sizeof(RowBest) + k * sizeof(Entry));
  return true;
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
                      static_cast<const uint64_t*>(b.finished), b.out_scores, b.out_parents, b.out_tokens};
  RowBest* rows = static_cast<RowBest*>(b.workspace);
  Entry* entries = reinterpret_cast<Entry*>(rows + (uint64_t)b.batch * b.beams);
  const dim3 grid(b.batch * b.beams);
  if (b.type == AGPU_ROW_F32) hipLaunchKernelGGL((beam_rows_kernel<float>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, rows, entries);
  else if (b.type == AGPU_ROW_F16) hipLaunchKernelGGL((beam_rows_kernel<f16_t>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, rows, entries);
  else hipLaunchKernelGGL((beam_rows_kernel<bf16_t>), grid, dim3(AGPU_BLOCK), 0, p->stream, a, rows, entries);
  AGPU_LAUNCH_CHECK();
  hipLaunchKernelGGL(beam_merge_kernel, dim3(b.batch), dim3(AGPU_BLOCK), 0, p->stream, a, rows, entries);
  AGPU_LAUNCH_CHECK();
  return AGPU_OK;
}

}  // extern "C"
