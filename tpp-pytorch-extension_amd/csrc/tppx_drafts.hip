// Which drafted tokens stand against the target's probabilities, and the token behind them.
//
// Nodes are packed as in the paged cache's operators: node 0 of a sequence is the token accepted last, the others are drafted, and row i
// of the logits is what the target says behind node i.  p = softmax(target / temperature) of a row (temperature 0: one for the first
// maximal logit).  From node 0 on, the children of a node are tried in order.  With candidates (no draft logits) child x stands where
//   u M < p(x),  M = 1 - the p of the siblings tried before it,
// and what is left of p for those behind it has no x.  With draft logits (chains: one child), q = softmax(draft / temperature) of the
// node's row, it stands where u q(x) < p(x), and leaves max(p - q, 0).  Where no child stands, the path ends and the next token is the
// first one whose cumulative sum of what is left exceeds `sample` times the whole sum.  Either way the tokens that come out are distributed
// as the target's own.  Everything in fp64: a token is a step function of these sums, and the sum of 10^5 terms in fp32 puts one draw in
// some 10^2 on the other side of a border.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "tppx_mx4.h"

namespace tppx {

struct DraftsParams {
  const int64_t* tokens;
  const void *target, *draft;
  const int32_t *cu, *parents;
  const float *uniforms, *sample, *temps;
  int32_t *path, *count;
  int64_t* next;
  int64_t t_ld, d_ld;
  int T, B, V;
  float temperature;
};

template <typename E>
__device__ __forceinline__ float logit(const E* row, int i) { // (what is no number is no token)
  float v;
  if constexpr (std::is_same_v<E, float>)
    v = row[i];
  else if constexpr (std::is_same_v<E, _Float16>)
    v = (float)row[i];
  else
    v = bf16_bits_to_f32(row[i]);
  return v == v ? v : -INFINITY;
}
// of a row: maximum, its first place, sum of the weights
struct RowStat {
  float top;
  int first;
  double sum;
};
// exp((x - top) / t); 1 at the maximum also where that is infinite, and t 0: nothing else
__device__ __forceinline__ double weight_of(float x, float top, double inv) {
  return x == top ? 1.0 : inv == 0.0 ? 0.0 : exp(((double)x - (double)top) * inv);
}

constexpr int DRAFT_THREADS = 1024;

template <typename E>
__global__ void __launch_bounds__(DRAFT_THREADS)
verify_kernel(const DraftsParams p) {
  __shared__ double red[DRAFT_THREADS];
  __shared__ float redf[DRAFT_THREADS];
  __shared__ int redi[DRAFT_THREADS];
  const int tid = threadIdx.x, b = (int)blockIdx.x;
  const int first = p.cu ? p.cu[b] : b, n = p.cu ? min(p.cu[b + 1], p.T) - first : 1;
  if (first < 0 || n < 1) {
    if (tid == 0) {
      p.count[b] = 0;
      p.next[b] = 0;
    }
    return;
  }
  const float temp = p.temps ? p.temps[b] : p.temperature;
  const double inv = temp > 0.f ? 1.0 / (double)temp : 0.0;
  const int32_t* const parents = p.parents ? p.parents + first : nullptr;
  auto sum_all = [&](double v) {
    red[tid] = v;
    __syncthreads();
    for (int s = DRAFT_THREADS / 2; s > 0; s /= 2) {
      if (tid < s)
        red[tid] += red[tid + s];
      __syncthreads();
    }
    const double r = red[0];
    __syncthreads();
    return r;
  };
  auto stat = [&](const E* row) {
    float top = -INFINITY;
    int at = p.V;
    for (int i = tid; i < p.V; i += DRAFT_THREADS) {
      const float x = logit(row, i);
      if (x > top || at == p.V) {
        top = x;
        at = i;
      }
    }
    redf[tid] = top;
    redi[tid] = at;
    __syncthreads();
    for (int s = DRAFT_THREADS / 2; s > 0; s /= 2) {
      if (tid < s) {
        const float x = redf[tid + s];
        const int j = redi[tid + s];
        if (j < p.V && (redi[tid] == p.V || x > redf[tid] || (x == redf[tid] && j < redi[tid]))) {
          redf[tid] = x;
          redi[tid] = j;
        }
      }
      __syncthreads();
    }
    RowStat r = {redf[0], redi[0], 0.0};
    __syncthreads();
    if (inv == 0.0) {
      r.sum = 1.0;
      return r;
    }
    double sum = 0.0;
    for (int i = tid; i < p.V; i += DRAFT_THREADS)
      sum += weight_of(logit(row, i), r.top, inv);
    r.sum = sum_all(sum);
    return r;
  };
  auto share = [&](const E* row, const RowStat& s, int64_t x) {
    if (x < 0 || x >= p.V)
      return 0.0;
    if (inv == 0.0)
      return x == s.first ? 1.0 : 0.0;
    return weight_of(logit(row, (int)x), s.top, inv) / s.sum;
  };
  int at = 0, len = 0;
  const E *prow, *qrow = nullptr;
  RowStat ps, qs;
  bool rejected = false;
  for (;;) {
    if (tid == 0)
      p.path[first + len] = at;
    len++;
    prow = (const E*)p.target + (int64_t)(first + at) * p.t_ld;
    ps = stat(prow);
    if (p.draft && inv != 0.0) {
      qrow = (const E*)p.draft + (int64_t)(first + at) * p.d_ld;
      qs = stat(qrow);
    }
    int down = -1;
    double left = 1.0;
    rejected = false;
    for (int c = at + 1; c < n && down < 0; c++) {
      const int up = parents ? parents[c] : c - 1;
      if (up != at)
        continue;
      const int64_t x = p.tokens[first + c];
      const double u = inv == 0.0 ? 0.0 : (double)p.uniforms[first + c];
      double px = share(prow, ps, x);
      if (qrow) {
        if (u * share(qrow, qs, x) < px)
          down = c;
      } else {
        for (int e = at + 1; e < c; e++) // (a sibling's token again: nothing is left of it)
          if ((parents ? parents[e] : e - 1) == at && p.tokens[first + e] == x)
            px = 0.0;
        if (u * left < px)
          down = c;
        left -= px;
      }
      rejected |= down < 0;
    }
    if (down < 0)
      break;
    at = down;
  }
  // What is left of the row, in order: each thread a run of it.
  auto rest = [&](int i, bool all) {
    const double w = share(prow, ps, i);
    if (all || !rejected)
      return w;
    if (qrow)
      return fmax(w - share(qrow, qs, i), 0.0);
    for (int c = at + 1; c < n; c++)
      if ((parents ? parents[c] : c - 1) == at && p.tokens[first + c] == i)
        return 0.0;
    return w;
  };
  const int per = (p.V + DRAFT_THREADS - 1) / DRAFT_THREADS, from = min(tid * per, p.V), to = min(from + per, p.V);
  bool all = false;
  double mine = 0.0;
  for (int i = from; i < to; i++)
    mine += rest(i, false);
  double whole = sum_all(mine);
  if (!(whole > 0.0)) {
    all = true;
    mine = 0.0;
    for (int i = from; i < to; i++)
      mine += rest(i, true);
    whole = sum_all(mine);
  }
  red[tid] = mine;
  __syncthreads();
  double before = 0.0;
  for (int t = 0; t < tid; t++)
    before += red[t];
  const double border = (inv == 0.0 ? 0.0 : (double)p.sample[b]) * whole;
  int found = p.V, last = -1;
  double run = before;
  for (int i = from; i < to; i++) {
    const double w = rest(i, all);
    run += w;
    if (w > 0.0)
      last = i;
    if (run > border && found == p.V)
      found = i;
  }
  redi[tid] = found;
  __syncthreads();
  if (tid == 0) {
    int r = p.V;
    for (int t = 0; t < DRAFT_THREADS; t++)
      r = min(r, redi[t]);
    redi[0] = r;
  }
  __syncthreads();
  const int r = redi[0];
  __syncthreads();
  redi[tid] = last;
  __syncthreads();
  if (tid == 0) {
    int z = 0;
    for (int t = 0; t < DRAFT_THREADS; t++)
      z = max(z, redi[t]);
    p.next[b] = r < p.V ? r : z;
    p.count[b] = len;
  }
  for (int i = len + tid; i < n; i += DRAFT_THREADS)
    p.path[first + i] = -1;
}

} // namespace tppx

using namespace tppx;

extern "C" int tppx_verify_drafts(const void* tokens, const void* target, const void* draft, int dtype, const void* cu, const void* parents,
                                  const void* uniforms, const void* sample, const void* temperatures, float temperature, void* path,
                                  void* count, void* next, int64_t T, int64_t B, int64_t V, int64_t t_ld, int64_t d_ld, void* ws,
                                  int64_t ws_bytes, tppx_stream_t stream) {
  const char* who = "tppx_verify_drafts";
  TPPX_REQUIRE(tokens && target && path && count && next, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(dtype == TPPX_DT_F32 || dtype == TPPX_DT_BF16 || dtype == TPPX_DT_F16, TPPX_EINVAL, "%s: dtype %d", who, dtype);
  const uintptr_t size = dtype == TPPX_DT_F32 ? 4 : 2;
  TPPX_REQUIRE((((uintptr_t)tokens | (uintptr_t)next) & 7u) == 0 && (((uintptr_t)target | (uintptr_t)draft) & (size - 1)) == 0 &&
                   (((uintptr_t)cu | (uintptr_t)parents | (uintptr_t)uniforms | (uintptr_t)sample | (uintptr_t)temperatures | (uintptr_t)path | (uintptr_t)count) & 3u) == 0,
               TPPX_EINVAL, "%s: pointer not aligned to its type", who);
  TPPX_REQUIRE(temperatures || (temperature >= 0.f && temperature < INFINITY), TPPX_EINVAL, "%s: temperature %g", who, (double)temperature);
  TPPX_REQUIRE((uniforms && sample) || (!temperatures && temperature == 0.f), TPPX_EINVAL, "%s: sampling needs random numbers", who);
  TPPX_REQUIRE(!draft || !parents, TPPX_EUNSUPPORTED, "%s: draft logits are taken for chains, without parents", who);
  TPPX_REQUIRE(T >= 0 && T < ((int64_t)1 << 30) && B > 0 && B < ((int64_t)1 << 24) && V > 0 && V < ((int64_t)1 << 30), TPPX_ESHAPE,
               "%s: bad shape T=%ld B=%ld V=%ld", who, (long)T, (long)B, (long)V);
  TPPX_REQUIRE(t_ld >= V && (!draft || d_ld >= V), TPPX_ESHAPE, "%s: row strides must hold a row", who);
  TPPX_REQUIRE(cu || T == B, TPPX_ESHAPE, "%s: %ld tokens of %ld sequences need their bounds", who, (long)T, (long)B);
  TPPX_REQUIRE(ws_bytes >= 0 && (ws_bytes == 0 || ws), TPPX_EINVAL, "%s: size given with a null pointer", who);
  DraftsParams p;
  memset(&p, 0, sizeof(p));
  p.tokens = (const int64_t*)tokens; p.target = target; p.draft = draft; p.cu = (const int32_t*)cu; p.parents = (const int32_t*)parents;
  p.uniforms = (const float*)uniforms; p.sample = (const float*)sample; p.temps = (const float*)temperatures; p.temperature = temperature;
  p.path = (int32_t*)path; p.count = (int32_t*)count; p.next = (int64_t*)next;
  p.t_ld = t_ld; p.d_ld = d_ld; p.T = (int)T; p.B = (int)B; p.V = (int)V;
  const dim3 grid((unsigned)B);
  if (dtype == TPPX_DT_F32)
    verify_kernel<float><<<grid, dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
  else if (dtype == TPPX_DT_F16)
    verify_kernel<_Float16><<<grid, dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
  else
    verify_kernel<uint16_t><<<grid, dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
  return check_hip(hipGetLastError(), who);
}

extern "C" int64_t tppx_verify_drafts_bytes(int64_t T, int64_t B, int64_t V, int drafts) {
  return 0;
}
