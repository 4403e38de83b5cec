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

// Two launches, three with draft logits.  The first goes over all logits, in pieces: maximum, its place, and the sum of the weights relative
// to that maximum.  The second decides for all nodes at once what u M and u q are compared with, walks from node 0 down, and finds the
// next token: the piece in which the border lies by the pieces' sums less the tried siblings' shares, then the token in it.  With draft
// logits max(p - q, 0) of the last row is a pass of its own over pieces, the second launch, and the third one finds the token.
struct DraftsParams {
  const int64_t* tokens;
  const void *target, *draft;
  const int32_t *cu, *parents;
  const float *uniforms, *sample, *temps;
  int32_t *path, *count;
  int64_t* next;
  struct Piece* pieces; // [sides][T][C]
  double* sums;         // [B][C] of what is left of a sequence's last row
  double *px, *qx;      // [T]
  int64_t t_ld, d_ld;
  int T, B, V, C, sides;
  float temperature;
};
struct Piece {
  double sum;
  float top;
  int first;
};
constexpr double LOG2E_64 = 1.4426950408889634;

// 2^y for y <= 0, 1e-15 relative: 2^f, f in [-1/2, 1/2], by its interpolation at the Chebyshev points of degree 10
__device__ __forceinline__ double exp2_64(double y) {
  y = fmax(y, -1100.0); // (below any double)
  const double n = __builtin_rint(y), f = y - n;
  double r = 7.072585489423359e-09;
  r = fma(r, f, 1.0208690645080226e-07);
  r = fma(r, f, 1.3215442588981224e-06);
  r = fma(r, f, 1.525265725816688e-05);
  r = fma(r, f, 0.00015403530441732765);
  r = fma(r, f, 0.0013333558230168993);
  r = fma(r, f, 0.009618129107606902);
  r = fma(r, f, 0.05550410866444769);
  r = fma(r, f, 0.24022650695910097);
  r = fma(r, f, 0.69314718055995);
  r = fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)n);
}
// the weight of a logit under the row's maximum: 1 for that, also where it is infinite; to2: log2 e / temperature, 0: nothing else
__device__ __forceinline__ double weight_of(float x, float top, double to2) {
  const double w = to2 == 0.0 ? 0.0 : exp2_64(((double)x - (double)top) * to2);
  return x == top ? 1.0 : w;
}
template <typename E>
__device__ __forceinline__ float logit_of(E v) { // (what is no number is no token)
  float x;
  if constexpr (std::is_same_v<E, uint16_t>)
    x = bf16_bits_to_f32(v);
  else
    x = (float)v;
  return x == x ? x : -INFINITY;
}
// 0: the first maximum alone (for what is no positive finite temperature, too)
__device__ __forceinline__ double to2_of(const DraftsParams& p, int b) {
  const float t = p.temps ? p.temps[b] : p.temperature;
  return t > 0.f && t < INFINITY ? LOG2E_64 / (double)t : 0.0;
}

constexpr int DRAFT_THREADS = 256;
// logits per 16 bytes
template <typename E>
constexpr int per16() { return 16 / (int)sizeof(E); }
// `n` logits of a row from `at` on, -inf behind its end (rows need no more than their type's alignment)
template <typename E>
__device__ __forceinline__ void load_logits(const E* row, int at, int V, float (&x)[per16<E>()]) {
  constexpr int N = per16<E>();
  if (at + N <= V) {
    E v[N];
    __builtin_memcpy(v, row + at, 16);
#pragma unroll
    for (int e = 0; e < N; e++)
      x[e] = logit_of(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; e++)
      x[e] = at + e < V ? logit_of(row[min(at + e, V - 1)]) : -INFINITY;
  }
}

template <int N, typename F>
__device__ __forceinline__ double reduce_lanes(double v, F&& f) {
#pragma unroll
  for (int d = 1; d < N; d *= 2)
    v = f(v, __shfl_xor(v, d));
  return v;
}

// ---------------------------------------------------------------------------
// All rows, a workgroup for a piece of 256 NV vectors of 16 bytes.
// ---------------------------------------------------------------------------
template <typename E, int NV>
__global__ void __launch_bounds__(DRAFT_THREADS)
draft_rows_kernel(const DraftsParams p) {
  constexpr int N = per16<E>();
  __shared__ float tops[4];
  __shared__ int firsts[4];
  __shared__ double sums[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = (int)(blockIdx.x / (unsigned)p.C), piece = (int)(blockIdx.x % (unsigned)p.C), side = (int)blockIdx.y;
  int b = 0;
  if (p.temps) {
    if (p.cu)
      b = min(sequence_of(p.cu, p.B, row), p.B - 1);
    else
      b = row;
  }
  const double to2 = to2_of(p, b);
  const E* const at = (const E*)(side ? p.draft : p.target) + (int64_t)row * (side ? p.d_ld : p.t_ld);
  const int from = piece * (DRAFT_THREADS * NV * N);
  float x[NV][N];
#pragma unroll
  for (int i = 0; i < NV; i++)
    load_logits<E>(at, from + (i * DRAFT_THREADS + tid) * N, p.V, x[i]);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int e = 0; e < N; e++)
      top = fmaxf(top, x[i][e]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
    top = fmaxf(top, __shfl_xor(top, d));
  int first = p.V;
  double sum = 0.0;
  if (to2 == 0.0) {
#pragma unroll
    for (int i = NV - 1; i >= 0; i--)
#pragma unroll
      for (int e = N - 1; e >= 0; e--) {
        const int j = from + (i * DRAFT_THREADS + tid) * N + e;
        first = x[i][e] == top && j < p.V ? j : first;
      }
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
      first = min(first, __shfl_xor(first, d));
  } else {
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < N; e++) { // (behind the end: -inf, which counts where the row is nothing else)
        const double w = weight_of(x[i][e], top, to2);
        sum += from + (i * DRAFT_THREADS + tid) * N + e < p.V ? w : 0.0;
      }
    sum = reduce_lanes<64>(sum, [](double a, double z) { return a + z; });
  }
  if (lane == 0) {
    tops[wave] = top;
    firsts[wave] = first;
    sums[wave] = sum;
  }
  __syncthreads();
  if (tid == 0) {
    Piece r = {0.0, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), p.V};
    for (int w = 3; w >= 0; w--) {
      if (sums[w] > 0.0)
        r.sum += sums[w] * weight_of(tops[w], r.top, to2);
      if (firsts[w] < p.V && tops[w] == r.top)
        r.first = firsts[w];
    }
    p.pieces[((int64_t)side * p.T + row) * p.C + piece] = r;
  }
}

// ---------------------------------------------------------------------------
// The walk and the next token.  LAST: finds the token; otherwise sums what is left of the last row's piece blockIdx.y.
// ---------------------------------------------------------------------------
constexpr int DRAFT_NODES = 256; // nodes of a sequence that are held in LDS; more go through the workspace
struct RowSum {
  double sum;
  float top;
  int first;
};

template <typename E, int NV, bool LAST>
__global__ void __launch_bounds__(DRAFT_THREADS)
draft_walk_kernel(const DraftsParams p) {
  constexpr int N = per16<E>(), PIECE = DRAFT_THREADS * NV * N;
  __shared__ double px_lds[DRAFT_NODES], qx_lds[DRAFT_NODES];
  __shared__ double tried_px[DRAFT_NODES]; // the last node's children: shares, pieces that their tokens lie in
  __shared__ int tried_in[DRAFT_NODES];
  __shared__ uint32_t gone[PIECE / 32]; // tokens of a piece that were tried
  __shared__ double red[DRAFT_THREADS];
  __shared__ int found_at[4];
  __shared__ int walk_at, walk_len, walk_tried, piece_at;
  __shared__ double piece_before, piece_border;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = (int)blockIdx.x;
  const int first = p.cu ? min(max(p.cu[b], 0), p.T) : b, n = p.cu ? min(p.cu[b + 1], p.T) - first : 1;
  if (n < 1) {
    if (LAST && tid == 0) {
      p.count[b] = 0;
      p.next[b] = 0;
    }
    return;
  }
  const double to2 = to2_of(p, b);
  const bool drawn = p.draft && to2 != 0.0;
  const int32_t* const parents = p.parents ? p.parents + first : nullptr;
  const int64_t* const tokens = p.tokens + first;
  auto parent = [&](int i) { return parents ? parents[i] : i - 1; };
  // a row's state from its pieces: G lanes take them in turn
  auto row_sum = [&](int side, int row, int u, auto G_) {
    constexpr int G = decltype(G_)::value;
    const Piece* const at = p.pieces + ((int64_t)side * p.T + row) * p.C;
    RowSum r = {0.0, -INFINITY, p.V};
    for (int i = u; i < p.C; i += G) {
      const Piece z = at[i];
      if (z.top > r.top) {
        r.sum = r.sum > 0.0 ? r.sum * weight_of(r.top, z.top, to2) : 0.0;
        r.top = z.top;
        r.first = z.first;
      } else if (z.top == r.top) {
        r.first = min(r.first, z.first);
      }
      if (z.sum > 0.0) // (a piece of nothing but -inf counts where the row is nothing else)
        r.sum += z.sum * weight_of(z.top, r.top, to2);
    }
#pragma unroll
    for (int d = 1; d < G; d *= 2) {
      const float top = __shfl_xor(r.top, d);
      const int place = __shfl_xor(r.first, d);
      const double sum = __shfl_xor(r.sum, d);
      const float both = fmaxf(r.top, top);
      r.first = top > r.top ? place : top == r.top ? min(r.first, place) : r.first;
      // (the same order in both lanes: their sums must not differ)
      const double a = r.sum * weight_of(r.top, both, to2), z = sum * weight_of(top, both, to2);
      r.sum = a + z;
      r.top = both;
    }
    return r;
  };
  auto share = [&](int side, int row, const RowSum& r, int64_t x) {
    if (x < 0 || x >= p.V)
      return 0.0;
    if (to2 == 0.0)
      return x == r.first ? 1.0 : 0.0;
    const E* const at = (const E*)(side ? p.draft : p.target) + (int64_t)row * (side ? p.d_ld : p.t_ld);
    return weight_of(logit_of(at[x]), r.top, to2) / r.sum;
  };
  // p (and q) of every node's token in its parent's row: 16 lanes a node
  double* const px = n <= DRAFT_NODES ? px_lds : p.px + first;
  double* const qx = n <= DRAFT_NODES ? qx_lds : p.qx + first;
  for (int i0 = 0; i0 < n; i0 += DRAFT_THREADS / 16) {
    const int i = i0 + tid / 16, u = tid % 16;
    const int up = i < n ? parent(i) : -1;
    if (up >= 0 && up < i) {
      const double a = share(0, first + up, row_sum(0, first + up, u, std::integral_constant<int, 16>{}), tokens[i]);
      const double z = drawn ? share(1, first + up, row_sum(1, first + up, u, std::integral_constant<int, 16>{}), tokens[i]) : 0.0;
      if (u == 0) {
        px[i] = a;
        if (drawn)
          qx[i] = z;
      }
    }
  }
  __syncthreads();
  if (wave == 0) { // down, all lanes alike
    int at = 0, len = 0, tried;
    for (;;) {
      if (LAST && lane == 0)
        p.path[first + len] = at;
      len++;
      int down = -1;
      double left = 1.0;
      tried = 0;
      for (int c0 = at + 1; c0 < n && down < 0; c0 += 64) {
        if (!parents && c0 > at + 1)
          break; // (a chain: one child)
        const int mine = c0 + lane;
        uint64_t children = __builtin_amdgcn_ballot_w64(mine < n && parent(mine) == at);
        while (children && down < 0) {
          const int c = c0 + __builtin_ctzll(children);
          children &= children - 1;
          const double u = to2 == 0.0 ? 0.0 : (double)p.uniforms[first + c];
          double x = px[c];
          if (drawn) {
            if (u * qx[c] < x)
              down = c;
          } else {
            bool again = false; // (nothing is left of a token that was tried)
            for (int e0 = at + 1; e0 < c; e0 += 64)
              again |= __builtin_amdgcn_ballot_w64(e0 + lane < c && parent(e0 + lane) == at && tokens[e0 + lane] == tokens[c]) != 0;
            x = again ? 0.0 : x;
            if (u * left < x)
              down = c;
            left -= x;
            if (tried < DRAFT_NODES && lane == 0) {
              const bool inside = tokens[c] >= 0 && tokens[c] < p.V;
              tried_px[tried] = x;
              tried_in[tried] = inside ? (int)tokens[c] / PIECE : -1;
            }
          }
          tried += down < 0;
        }
      }
      if (down < 0)
        break;
      at = down;
    }
    if (lane == 0) {
      walk_at = at;
      walk_len = len;
      walk_tried = tried;
    }
  }
  __syncthreads();
  const int at = walk_at, len = walk_len;
  const int tried = walk_tried;
  const int row = first + at;
  if (LAST) {
    for (int i = len + tid; i < n; i += DRAFT_THREADS)
      p.path[first + i] = -1;
    if (tid == 0)
      p.count[b] = len;
  }
  const RowSum ps = row_sum(0, row, lane, std::integral_constant<int, 64>{});
  if (to2 == 0.0) {
    if (LAST && tid == 0)
      p.next[b] = ps.first;
    return;
  }
  const bool residual = drawn && tried;
  RowSum qs = {1.0, 0.f, 0};
  if (residual)
    qs = row_sum(1, row, lane, std::integral_constant<int, 64>{});
  const E* const prow = (const E*)p.target + (int64_t)row * p.t_ld;
  const E* const qrow = (const E*)p.draft + (int64_t)row * p.d_ld;
  // What is left of a vector of 16 bytes of the last row: p without the tokens that were tried, or max(p - q, 0).  all: p.
  auto mark = [&](int piece) { // the tried tokens of a piece
    if (!tried || drawn)
      return;
    for (int i = tid; i < PIECE / 32; i += DRAFT_THREADS)
      gone[i] = 0;
    __syncthreads();
    for (int c = at + 1 + tid; c < n; c += DRAFT_THREADS) {
      const int64_t x = parent(c) == at ? tokens[c] : -1;
      if (x >= 0 && x < p.V && x / PIECE == piece)
        atomicOr(&gone[x % PIECE / 32], 1u << (x % 32));
    }
    __syncthreads();
  };
  const double pn = 1.0 / ps.sum, qn = 1.0 / qs.sum;
  auto rest = [&](int from, bool all, double (&w)[N]) {
    float x[N], y[N];
    load_logits<E>(prow, from, p.V, x);
    if (residual && !all)
      load_logits<E>(qrow, from, p.V, y);
    const bool without = tried && !drawn && !all;
#pragma unroll
    for (int e = 0; e < N; e++) {
      w[e] = weight_of(x[e], ps.top, to2) * pn;
      if (residual && !all)
        w[e] = fmax(w[e] - weight_of(y[e], qs.top, to2) * qn, 0.0);
      if (without && gone[(from + e) % PIECE / 32] >> ((from + e) % 32) & 1)
        w[e] = 0.0;
      w[e] = from + e < p.V ? w[e] : 0.0;
    }
  };
  auto sum_of_piece = [&](int piece, bool all) { // in all threads; `gone` marked
    double s = 0.0;
    for (int i = 0; i < NV; i++) {
      double w[N];
      rest(piece * PIECE + (i * DRAFT_THREADS + tid) * N, all, w);
#pragma unroll
      for (int e = 0; e < N; e++)
        s += w[e];
    }
    s = reduce_lanes<64>(s, [](double a, double z) { return a + z; });
    __syncthreads();
    if (lane == 0)
      red[wave] = s;
    __syncthreads();
    s = (red[0] + red[1]) + (red[2] + red[3]);
    return s;
  };
  double* const sums = p.sums + (int64_t)b * p.C;
  if constexpr (!LAST) {
    if (residual) {
      const double s = sum_of_piece((int)blockIdx.y, false);
      if (tid == 0)
        sums[blockIdx.y] = s;
    }
    return;
  } else {
    // The pieces' sums: from the first launch less the tried tokens' shares (a difference of sums near 1, so a rest that small is
    // summed anew, as it is where more were tried than are kept), from the second one, or, where nothing is left, p.
    bool all = !tried;
    for (int round = 0;; round++) {
      if (wave == 0) {
        auto of_piece = [&](int i) {
          if (i >= p.C)
            return 0.0;
          if (!all && (drawn || round > 0))
            return sums[i];
          const Piece z = p.pieces[(int64_t)row * p.C + i];
          double s = z.sum > 0.0 ? z.sum * weight_of(z.top, ps.top, to2) * pn : 0.0;
          if (!all)
            for (int c = 0; c < min(tried, DRAFT_NODES); c++)
              s -= tried_in[c] == i ? tried_px[c] : 0.0;
          return fmax(s, 0.0);
        };
        const double head = of_piece(lane);
        double whole = 0.0;
        for (int i0 = 0; i0 < p.C; i0 += 64)
          whole += reduce_lanes<64>(i0 ? of_piece(i0 + lane) : head, [](double a, double z) { return a + z; });
        const double border = (double)p.sample[b] * whole;
        double before = 0.0, start = 0.0;
        int piece = -1, last = 0;
        for (int i0 = 0; i0 < p.C && piece < 0; i0 += 64) {
          const double s = i0 ? of_piece(i0 + lane) : head;
          double run = s;
#pragma unroll
          for (int d = 1; d < 64; d *= 2) {
            const double t = __shfl_up(run, d);
            run += lane >= d ? t : 0.0;
          }
          const uint64_t beyond = __builtin_amdgcn_ballot_w64(s > 0.0 && before + run > border);
          const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0);
          if (beyond) {
            const int j = __builtin_ctzll(beyond);
            piece = i0 + j;
            start = before + __shfl(run - s, j);
          } else if (some) { // (where the border is rounded past the last one)
            const int j = 63 - __builtin_clzll(some);
            last = i0 + j;
            start = before + __shfl(run - s, j);
          }
          before += __shfl(run, 63);
        }
        if (lane == 0) {
          piece_at = piece < 0 ? last : piece;
          piece_before = start;
          const bool anew = round == 0 && !all && !drawn;
          piece_border = whole > (anew ? 0x1p-30 : 0.0) && !(anew && tried > DRAFT_NODES) ? border : -1.0;
        }
      }
      __syncthreads();
      const bool fine = piece_border >= 0.0;
      __syncthreads();
      if (fine)
        break;
      if (all || drawn || round > 0) {
        if (all)
          break; // (does not happen: p sums to 1)
        all = true;
        continue;
      }
      for (int i = 0; i < p.C; i++) { // too little for differences
        mark(i);
        const double s = sum_of_piece(i, false);
        if (tid == 0)
          sums[i] = s;
      }
      __syncthreads();
    }
    // the token: a thread takes a run of the piece
    const int piece = piece_at;
    const double border = piece_border;
    mark(piece);
    constexpr int RUN = NV * N;
    double w[NV][N], s = 0.0;
#pragma unroll
    for (int i = 0; i < NV; i++) {
      rest(piece * PIECE + tid * RUN + i * N, all, w[i]);
#pragma unroll
      for (int e = 0; e < N; e++)
        s += w[i][e];
    }
    double run = s;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double t = __shfl_up(run, d);
      run += lane >= d ? t : 0.0;
    }
    if (lane == 63)
      red[wave] = run;
    __syncthreads();
    double before = piece_before;
    for (int i = 0; i < wave; i++)
      before += red[i];
    before += run - s;
    int found = p.V, last = -1;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < N; e++) {
        before += w[i][e];
        const int x = piece * PIECE + tid * RUN + i * N + e;
        if (w[i][e] > 0.0) {
          last = x;
          found = before > border && found == p.V ? x : found;
        }
      }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      found = min(found, __shfl_xor(found, d));
      last = max(last, __shfl_xor(last, d));
    }
    if (lane == 0)
      found_at[wave] = found;
    __syncthreads();
    found = min(min(found_at[0], found_at[1]), min(found_at[2], found_at[3]));
    __syncthreads();
    if (lane == 0)
      found_at[wave] = last;
    __syncthreads();
    if (tid == 0) // (a border that is rounded past the piece's last token: that one)
      p.next[b] = found < p.V ? found : max(max(max(found_at[0], found_at[1]), max(found_at[2], found_at[3])), 0);
  }
}

static int64_t draft_pieces(int64_t V, int64_t size, int nv) { return (V * size + DRAFT_THREADS * 16 * nv - 1) / (DRAFT_THREADS * 16 * nv); }
// vectors of 16 bytes that a thread takes of a row
static int draft_vectors(int64_t rows, int64_t V, int64_t size) {
  return rows * draft_pieces(V, size, 4) >= 512 ? 4 : 1;
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
  p.t_ld = t_ld; p.d_ld = d_ld; p.T = (int)T; p.B = (int)B; p.V = (int)V; p.sides = draft ? 2 : 1;
  const int nv = draft_vectors(T * p.sides, V, size);
  p.C = (int)draft_pieces(V, size, nv);
  TPPX_REQUIRE(T * p.C < ((int64_t)1 << 31) && p.C <= 65535, TPPX_ESHAPE, "%s: problem too large", who);
  const int64_t need = tppx_verify_drafts_bytes(T, B, V, draft != nullptr);
  TPPX_REQUIRE(ws && ws_bytes >= need, TPPX_EINVAL, "%s: needs %ld bytes of workspace, got %ld", who, (long)need, (long)ws_bytes);
  TPPX_REQUIRE(aligned16(ws), TPPX_EINVAL, "%s: workspace not 16-byte aligned", who);
  p.pieces = (Piece*)ws;
  p.sums = (double*)(p.pieces + p.sides * T * p.C);
  p.px = p.sums + B * p.C;
  p.qx = p.px + T;
  auto go = [&](auto e, auto nv_) {
    using E = decltype(e);
    constexpr int NV = decltype(nv_)::value;
    if (T > 0)
      draft_rows_kernel<E, NV><<<dim3((unsigned)(T * p.C), (unsigned)p.sides), dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
    if (T > 0 && draft)
      draft_walk_kernel<E, NV, false><<<dim3((unsigned)B, (unsigned)p.C), dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
    draft_walk_kernel<E, NV, true><<<dim3((unsigned)B), dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
  };
  auto typed = [&](auto e) {
    if (nv == 4)
      go(e, std::integral_constant<int, 4>{});
    else
      go(e, std::integral_constant<int, 1>{});
  };
  if (dtype == TPPX_DT_F32)
    typed(float{});
  else if (dtype == TPPX_DT_F16)
    typed(_Float16{});
  else
    typed(uint16_t{});
  return check_hip(hipGetLastError(), who);
}

extern "C" int64_t tppx_verify_drafts_bytes(int64_t T, int64_t B, int64_t V, int drafts) {
  // (of the type with the most pieces, in the form with the most)
  const int64_t C = draft_pieces(V, 4, 1);
  return (drafts ? 2 : 1) * T * C * (int64_t)sizeof(Piece) + B * C * 8 + 2 * T * 8 + 256;
}
