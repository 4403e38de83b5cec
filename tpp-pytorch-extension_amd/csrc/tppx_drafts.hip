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

// Two launches.  The first goes over all logits, in pieces: maximum, its place, and the sum of the weights relative to that maximum.  The
// second decides for all nodes at once what u M and u q are compared with, walks from node 0 down, and finds the next token: the piece in
// which the border lies by the pieces' sums less the tried siblings' shares, then the token in it.  With draft logits max(p - q, 0) of the
// last row is summed by a workgroup for each piece, and the one that ends last finds the token.  Small problems without draft logits are one
// launch, in which the workgroup that leaves a sequence's last piece goes on with the walk.
struct Piece {
  double sum;
  float top;
  int first;
};
typedef Piece RowSum;
struct NodeShare { // of a node's token in its parent's row
  double px, qx;
  int up, token;
  float u;
};
struct Walk {
  RowSum p, q; // of the last node's row
  int at, len, tried;
};
struct DraftsParams {
  const int64_t* tokens;
  const void *target, *draft;
  const int32_t *cu, *parents;
  const float *uniforms, *sample, *temps;
  int32_t *path, *count;
  int64_t* next;
  Piece* pieces;    // [sides][T][C]
  double* sums;     // [B][C] of what is left of a sequence's last row
  unsigned int* ended; // [B] workgroups that have summed their piece of it, from 0 in the first launch
  unsigned int* left;  // pieces that a sequence has, DRAFT_STRIDE apart; 0 between launches.  Null: two launches
  RowSum* rows;     // [2][T], of sequences too long for LDS
  NodeShare* nodes; // [T], of those
  int64_t t_ld, d_ld;
  int T, B, V, C, sides;
  double to2; // of the temperature, where that is a number
};
constexpr int DRAFT_STRIDE = 64;
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
// The same for many: 2^(x k) = 2^(n / 256) 2^(f / 256), n whole, f in [-1/2, 1/2]; the first from a table, the second by an
// interpolation of degree 3, 4e-14 relative.  Eight instructions in 64 bits where the polynomial takes nineteen.  The sum is relative to
// 2^(r / 256), r the whole number next to that of the maximum, so that no difference is taken.  `lowest` stands for what lies below
// it (its weight is 2^-900).  A NaN may come out for one that comes in.
struct Powers { // 2^(j / 256), less the bits that n << 12 adds to it
  double v[256];
  constexpr Powers() : v() {
    constexpr double f[8] = {1.0027112750502025, 1.0054299011128027, 1.0108892860517005, 1.0218971486541166, 1.0442737824274138, 1.0905077326652577, 1.189207115002721, 1.4142135623730951};
    for (int j = 0; j < 256; j++) {
      double x = 1.0;
      for (int i = 0; i < 8; i++)
        x *= j >> i & 1 ? f[i] : 1.0;
      v[j] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, x) - ((uint64_t)j << 44));
    }
  }
};
__device__ constexpr Powers POWERS;
struct ManyWeights {
  const double* table;
  double k, magic;
  float lowest;
  __device__ __forceinline__ ManyWeights(const double* t, float top, double to2)
      : table(t), k(to2 * 256.0), magic(0x1.8p52 - __builtin_rint((double)top * (to2 * 256.0))), lowest(top - 900.0f * __builtin_amdgcn_rcpf((float)to2)) {}
  static __device__ __forceinline__ bool fits(float top, double to2) { return fabsf(top) < 1e5f && to2 < 64.0 && to2 > 1e-6 && fabsf(top) * (float)to2 < 1e6f; }
  // what the sum of the weights relative to the maximum is that of these times, and its logarithm
  __device__ __forceinline__ double log_off(float top) const { return ((0x1.8p52 - magic) - (double)top * k) * (1.0 / 256.0); }
  __device__ __forceinline__ double off(float top) const { return exp2_64(log_off(top)); }
  // 2^(n / 256), and what is left
  __device__ __forceinline__ double parts(float x, double& g) const {
    float c;
    asm("v_max_f32 %0, %1, %2" : "=v"(c) : "v"(x), "v"(lowest));
    const double d = (double)c, t = fma(d, k, magic), f = fma(d, k, magic - t); // (t is rounded to a whole number, which its low bits are)
    const int n = __double2loint(t);
    const double a = table[n & 255];
    g = fma(f, fma(f, fma(f, 3.3083029079191157e-09, 3.665566016796724e-06), 0.0027076061740622863), 1.0);
    return __hiloint2double(__double2hiint(a) + (n << 12), __double2loint(a));
  }
  template <int N>
  __device__ __forceinline__ double sum(const float (&x)[N], double s) const {
#pragma unroll
    for (int e = 0; e < N; e++) {
      double g;
      const double w = parts(x[e], g);
      s = fma(w, g, s);
    }
    return s;
  }
  __device__ __forceinline__ double operator()(float x) const { // (below `lowest` nothing: no token of that weight is drawn)
    double g;
    const double w = parts(x, g);
    return x > lowest ? w * g : 0.0;
  }
};
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
  if (!p.temps)
    return p.to2;
  const float t = p.temps[b];
  return t > 0.f && t < INFINITY ? LOG2E_64 / (double)t : 0.0;
}

constexpr int DRAFT_THREADS = 256;
// logits per 16 bytes
template <typename E>
constexpr int per16() { return 16 / (int)sizeof(E); }
// logits as they lie in 16 bytes
template <typename E>
__device__ __forceinline__ void raw_logits(const uint4& v, float (&x)[per16<E>()]) {
  const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (std::is_same_v<E, float>) {
      x[i] = __uint_as_float(d[i]);
    } else if constexpr (std::is_same_v<E, uint16_t>) {
      x[2 * i] = __uint_as_float(d[i] << 16);
      x[2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u);
    } else {
      x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)d[i]);
      x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(d[i] >> 16));
    }
  }
}
// 16 bytes of a row from logit `at` on, -inf behind its end (rows need no more than their type's alignment)
template <typename E>
__device__ __forceinline__ uint4 load_raw(const E* row, int at, int V) {
  constexpr int N = per16<E>();
  constexpr uint32_t none = std::is_same_v<E, float> ? 0xff800000u : std::is_same_v<E, uint16_t> ? 0xff80ff80u : 0xfc00fc00u;
  uint4 v = make_uint4(none, none, none, none);
  if (at + N <= V) {
    __builtin_memcpy(&v, row + at, 16);
  } else if (at < V) {
    uint32_t d[4] = {none, none, none, none};
#pragma unroll
    for (int e = 0; e < N; e++)
      if (at + e < V) {
        if constexpr (N == 4)
          d[e] = __builtin_bit_cast(uint32_t, row[at + e]);
        else
          d[e / 2] = e & 1 ? (d[e / 2] & 0xffffu) | (uint32_t)__builtin_bit_cast(uint16_t, row[at + e]) << 16
                           : (d[e / 2] & 0xffff0000u) | __builtin_bit_cast(uint16_t, row[at + e]);
      }
    v = make_uint4(d[0], d[1], d[2], d[3]);
  }
  return v;
}
// N logits from `at` on
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

__device__ __forceinline__ double add64(double a, double z) { return a + z; }
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lane(double v) { // (0 where there is no such lane)
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, ROWS == 0xf);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, ROWS == 0xf);
  return __hiloint2double(hi, lo);
}
// sum over the lanes below, and this one's; all lanes take part
__device__ __forceinline__ double scan64(double v) {
  v += from_lane<0x111, 0xf>(v); // row_shr:1
  v += from_lane<0x112, 0xf>(v);
  v += from_lane<0x114, 0xf>(v);
  v += from_lane<0x118, 0xf>(v);
  v += from_lane<0x142, 0xa>(v); // row_bcast:15 into the second and the last row
  v += from_lane<0x143, 0xc>(v); // row_bcast:31 into the upper rows
  return v;
}

// the largest of a wave, in all lanes
__device__ __forceinline__ float top_of_wave(float v) {
  auto step = [&](auto c, auto r) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), decltype(c)::value, decltype(r)::value, 0xf, false)));
  };
  constexpr std::integral_constant<int, 15> all{};
  step(std::integral_constant<int, 0x111>{}, all);
  step(std::integral_constant<int, 0x112>{}, all);
  step(std::integral_constant<int, 0x114>{}, all);
  step(std::integral_constant<int, 0x118>{}, all);
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 10>{});
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 12>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
template <int N, typename F>
__device__ __forceinline__ double reduce_lanes(double v, F&& f) {
#pragma unroll
  for (int d = 1; d < N; d *= 2)
    v = f(v, __shfl_xor(v, d));
  return v;
}

// ---------------------------------------------------------------------------
// All rows, a workgroup for a piece of 256 NV vectors of 16 bytes.  Bound by instruction issue: 402 rows of 152000 bf16 logits (122 MB) 34 us,
// 3.6 TB/s, of which 26 are the 531 vector instructions for 32 logits of every thread (12.5 a logit, 8 of those in 64 bits).  At a temperature
// 0, without sums, 26 us, 4.6 TB/s.
// ---------------------------------------------------------------------------
// The piece, in thread 0.
template <typename E, int NV>
__device__ __forceinline__ Piece piece_of_row(const DraftsParams& p, int b, int row, int piece, int side) {
  constexpr int N = per16<E>();
  __shared__ float tops[4];
  __shared__ int firsts[4];
  __shared__ double sums[4], offs[4]; // of a wave, relative to 2^off times the weight of its maximum
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double to2 = to2_of(p, b);
  const E* const at = (const E*)(side ? p.draft : p.target) + (int64_t)row * (side ? p.d_ld : p.t_ld);
  const int from = piece * (DRAFT_THREADS * NV * N);
  int first = p.V;
  double sum = 0.0, off = 0.0;
  float top = -INFINITY;
  bool done = false; // (uniform in a wave)
  if (NV > 1 && to2 != 0.0) {
    __shared__ double table[256];
    uint4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; i++)
      v[i] = load_raw<E>(at, from + (i * DRAFT_THREADS + tid) * N, p.V);
    table[tid] = POWERS.v[tid];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float x[N];
      raw_logits<E>(v[i], x);
#pragma unroll
      for (int e = 0; e < N; e += 2)
        asm("v_max3_f32 %0, %0, %1, %2" : "+v"(top) : "v"(x[e]), "v"(x[e + 1]));
    }
    top = top_of_wave(top);
    if (from + wave * (64 * N) >= p.V) { // (behind the end)
      done = true;
    } else if (ManyWeights::fits(top, to2)) {
      const ManyWeights many(table, top, to2);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        float x[N];
        raw_logits<E>(v[i], x);
        sum = many.sum(x, sum);
      }
      sum = __shfl(scan64(sum), 63);
      off = many.log_off(top);
      done = sum > 0.0; // (and no NaN)
    }
  }
  if (!done) {
    float x[NV][N];
#pragma unroll
    for (int i = 0; i < NV; i++)
      load_logits<E>(at, from + (i * DRAFT_THREADS + tid) * N, p.V, x[i]);
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < N; e++)
        top = fmaxf(top, x[i][e]);
    top = top_of_wave(top);
    sum = off = 0.0;
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
      sum = __shfl(scan64(sum), 63);
    }
  }
  if (lane == 0) {
    tops[wave] = top;
    firsts[wave] = first;
    sums[wave] = sum;
    offs[wave] = off;
  }
  __syncthreads();
  // lanes 0 to 3: a wave's each
  const int w = tid & 3;
  const float most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), mine = tops[w];
  double v = sums[w];
  if (tid < 64 && to2 != 0.0)
    v = v > 0.0 ? v * exp2_64(mine == most ? offs[w] : ((double)mine - (double)most) * to2 + offs[w]) : 0.0;
  int place = firsts[w] < p.V && mine == most ? firsts[w] : p.V;
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    v += __shfl_xor(v, d);
    place = min(place, __shfl_xor(place, d));
  }
  return Piece{v, most, place};
}

template <typename E, int NV>
__global__ void __launch_bounds__(DRAFT_THREADS)
draft_rows_kernel(const DraftsParams p) {
  const int tid = threadIdx.x, row = (int)blockIdx.x, piece = (int)blockIdx.y, side = (int)blockIdx.z;
  int b = 0;
  if (p.temps || side) {
    b = p.cu ? sequence_of(p.cu, p.B, row) : row;
    if (side && (!p.cu || b >= p.B || p.cu[b + 1] == row + 1))
      return; // (nothing was drawn from the last node's)
    b = min(b, p.B - 1);
  }
  if (side == 0 && row == 0 && piece == 0 && p.sides == 2)
    for (int i = tid; i < p.B; i += DRAFT_THREADS)
      p.ended[i] = 0;
  const Piece r = piece_of_row<E, NV>(p, b, row, piece, side);
  if (tid == 0)
    p.pieces[((int64_t)side * p.T + row) * p.C + piece] = r;
}

// ---------------------------------------------------------------------------
// The walk and the next token, a workgroup for a sequence: the state of its rows from their pieces, every node's token's p (and q)
// in its parent's row, then down.  DRAFTS: a workgroup for each piece (blockIdx.y) walks down, sums what is left of its piece of the last
// row, and the one that ends last goes on to the token (nobody waits for another one).
// What they spend is waiting: row sums, nodes, the way down, the pieces and the token are five trips to memory or LDS one after another.
// 5 nodes, greedy 3.2 us; 10 trees of up to 60 nodes 12.2; 24 drawn chains 20, of which the token is
// 7 (with a launch of its own for that 13.3 + 8.5).
// ---------------------------------------------------------------------------
constexpr int DRAFT_NODES = 256; // nodes of a sequence that are held in LDS; more go through the workspace
// threads of a workgroup: where there is one for each piece, few enough that all of them run at once (24 chains' sums of 128000 logits alone
// 13.3 us, with 1024 threads 17.4)
constexpr int walk_threads(bool drafts) { return drafts ? 512 : 1024; }

template <bool SHARED>
__device__ __forceinline__ Piece load_piece(const Piece* at) {
  if constexpr (!SHARED)
    return *at;
  const uint64_t* const w = reinterpret_cast<const uint64_t*>(at);
  const uint64_t s = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), z = __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return Piece{__builtin_bit_cast(double, s), __uint_as_float((uint32_t)z), (int)(z >> 32)};
}
// first row and nodes of a sequence (fewer than 1: none)
__device__ __forceinline__ void bounds_of(const DraftsParams& p, int b, int& first, int& n) {
  first = p.cu ? min(max(p.cu[b], 0), p.T) : b;
  n = p.cu ? min(max(p.cu[b + 1], 0), p.T) - first : 1;
}
// SHARED: pieces of the same launch, from the level that all XCDs share
template <typename E, int NV, bool DRAFTS, int THREADS, bool SHARED>
__device__ __forceinline__ void walk_sequence(const DraftsParams& p, int b) {
  constexpr int N = per16<E>(), PIECE = DRAFT_THREADS * NV * N, WAVES = THREADS / 64;
  constexpr int VECTORS = DRAFT_THREADS * NV, EACH = VECTORS > THREADS ? VECTORS / THREADS : 1; // of a piece, of a thread
  __shared__ RowSum rows_lds[2][DRAFT_NODES];
  __shared__ NodeShare nodes_lds[DRAFT_NODES];
  __shared__ double tried_px[DRAFT_NODES]; // the last node's children: shares, pieces that their tokens lie in
  __shared__ int tried_in[DRAFT_NODES];
  __shared__ uint32_t gone[PIECE / 32]; // tokens of a piece that were tried
  __shared__ double red[WAVES];
  __shared__ int found_at[WAVES], last_at[WAVES];
  __shared__ double table[256];
  __shared__ Walk walk;
  __shared__ int piece_at, ended_last;
  __shared__ double piece_before, piece_border;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool lead = !DRAFTS || blockIdx.y == 0;
  int first, n;
  bounds_of(p, b, first, n);
  if (n < 1) {
    if (lead && tid == 0) {
      p.count[b] = 0;
      p.next[b] = 0;
    }
    return;
  }
  const double to2 = to2_of(p, b);
  const bool drawn = DRAFTS && to2 != 0.0;
  const float sample = to2 != 0.0 ? p.sample[b] : 0.f;
  if (tid < 256)
    table[tid] = POWERS.v[tid]; // (read behind a barrier)
  const int32_t* const parents = p.parents ? p.parents + first : nullptr;
  const int64_t* const tokens = p.tokens + first;
  auto parent = [&](int i) { return parents ? parents[i] : i - 1; };
  auto logits = [&](int side, int row) { return (const E*)(side ? p.draft : p.target) + (int64_t)row * (side ? p.d_ld : p.t_ld); };

  {
    const bool small = n <= DRAFT_NODES;
    NodeShare* const nodes = small ? nodes_lds : p.nodes + first;
    RowSum* const prows = small ? rows_lds[0] : p.rows + first;
    RowSum* const qrows = small ? rows_lds[1] : p.rows + p.T + first;
    // a node's token and its logits in its parent's row: asked for while the rows are summed up
    auto own = [&](int i, NodeShare& z, float& x, float& y) {
      z.up = parent(i);
      z.up = z.up < i ? max(z.up, -1) : -1;
      const int64_t t = tokens[i];
      z.token = t >= 0 && t < p.V ? (int)t : -1;
      z.u = p.uniforms && to2 != 0.0 ? p.uniforms[first + i] : 0.f;
      x = y = 0.f;
      if (z.up >= 0 && z.token >= 0) {
        x = logit_of(logits(0, first + z.up)[z.token]);
        if (drawn)
          y = logit_of(logits(1, first + z.up)[z.token]);
      }
    };
    // (the first piece of the first row, too: the loads from memory are what this launch waits for)
    const int sides = drawn ? 2 : 1, u = tid % 16;
    auto pieces_of = [&](int i) { return p.pieces + ((int64_t)(i >= n) * p.T + first + (i >= n ? i - n : i)) * p.C; };
    Piece ahead = {0.0, -INFINITY, p.V};
    if (tid / 16 < sides * n && u < p.C)
      ahead = load_piece<SHARED>(pieces_of(tid / 16) + u);
    NodeShare z0;
    float x0, y0;
    if (tid < n)
      own(tid, z0, x0, y0);
    // 16 lanes a row: its pieces in turn
    for (int i = tid / 16; i < sides * n; i += THREADS / 16) {
      const int side = i >= n, r = i - side * n;
      const Piece* const at = pieces_of(i);
      if (i != tid / 16)
        ahead = u < p.C ? load_piece<SHARED>(at + u) : Piece{0.0, -INFINITY, p.V};
      float top = ahead.top;
      int place = ahead.first;
      for (int c = u + 16; c < p.C; c += 16) {
        const Piece z = load_piece<SHARED>(at + c);
        const float t = z.top;
        const int f = z.first;
        place = t > top ? f : t == top ? min(place, f) : place;
        top = fmaxf(top, t);
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) {
        const float t = __shfl_xor(top, d);
        const int f = __shfl_xor(place, d);
        place = t > top ? f : t == top ? min(place, f) : place;
        top = fmaxf(top, t);
      }
      double sum = 0.0;
      if (to2 != 0.0) {
        sum = ahead.sum > 0.0 ? ahead.sum * weight_of(ahead.top, top, to2) : 0.0;
        for (int c = u + 16; c < p.C; c += 16) {
          const Piece z = load_piece<SHARED>(at + c);
          sum += z.sum > 0.0 ? z.sum * weight_of(z.top, top, to2) : 0.0;
        }
      }
      sum = reduce_lanes<16>(sum, add64);
      if (u == 0)
        (side ? qrows : prows)[r] = RowSum{sum, top, place};
    }
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      if (i != tid)
        own(i, z0, x0, y0);
      z0.px = z0.qx = 0.0;
      if (z0.up >= 0 && z0.token >= 0) {
        const RowSum r = prows[z0.up];
        z0.px = to2 == 0.0 ? (z0.token == r.first ? 1.0 : 0.0) : weight_of(x0, r.top, to2) / r.sum;
        if (drawn) {
          const RowSum s = qrows[z0.up];
          z0.qx = weight_of(y0, s.top, to2) / s.sum;
        }
      }
      nodes[i] = z0;
    }
    __syncthreads();
    if (parents) { // (nothing is left of a token that was tried before)
      for (int i = wave; i < n; i += WAVES) {
        const int up = nodes[i].up, token = nodes[i].token;
        bool again = false;
        for (int e = up + 1 + lane; e < i; e += 64)
          again |= nodes[e].up == up && nodes[e].token == token;
        if (__builtin_amdgcn_ballot_w64(again) != 0 && lane == 0)
          nodes[i].px = 0.0;
      }
      __syncthreads();
    }
    if (wave == 0) { // down, all lanes alike
      int at = 0, len = 0, tried = 0;
      if (!parents) { // a chain: the first node that does not stand ends it
        int end = n;
        for (int i0 = 0; i0 < n && end == n; i0 += 64) {
          const int i = i0 + lane;
          const NodeShare z = nodes[min(i, n - 1)];
          const bool fails = i > 0 && i < n && !((double)z.u * (drawn ? z.qx : 1.0) < z.px);
          const uint64_t bad = __builtin_amdgcn_ballot_w64(fails);
          if (bad)
            end = i0 + __builtin_ctzll(bad);
          if (lead)
            if (i < min(i0 + 64, n))
              p.path[first + i] = i < end ? i : -1;
        }
        at = end - 1;
        len = end;
        if (end < n) {
          tried = 1;
          if (lane == 0) {
            tried_px[0] = nodes[end].px;
            tried_in[0] = nodes[end].token < 0 ? -1 : nodes[end].token / PIECE;
          }
          if (lead)
            for (int i = end / 64 * 64 + 64 + lane; i < n; i += 64)
              p.path[first + i] = -1;
        }
      } else {
        for (;;) {
          if (lane == 0)
            p.path[first + len] = at;
          len++;
          int down = -1;
          double left = 1.0;
          tried = 0;
          for (int c0 = at + 1; c0 < n && down < 0; c0 += 64) {
            const int c = c0 + lane;
            const NodeShare z = nodes[min(c, n - 1)];
            const bool child = c < n && z.up == at;
            const double x = child ? z.px : 0.0, upto = scan64(x);
            const uint64_t children = __builtin_amdgcn_ballot_w64(child);
            const uint64_t stands = __builtin_amdgcn_ballot_w64(child && (double)z.u * (left - (upto - x)) < x);
            if (stands)
              down = c0 + __builtin_ctzll(stands);
            const int place = tried + __popcll(children & ((1ull << lane) - 1));
            if (!stands && child && place < DRAFT_NODES) {
              tried_px[place] = x;
              tried_in[place] = z.token < 0 ? -1 : z.token / PIECE;
            }
            tried += __popcll(children);
            left -= __shfl(upto, 63);
          }
          if (down < 0)
            break;
          at = down;
        }
        for (int i = len + lane; i < n; i += 64)
          p.path[first + i] = -1;
      }
      if (lane == 0)
        walk = Walk{prows[at], drawn ? qrows[at] : RowSum{1.0, 0.f, 0}, at, len, tried};
    }
    __syncthreads();
  }
  const int at = walk.at, tried = walk.tried, row = first + at;
  if (lead && tid == 0)
    p.count[b] = walk.len;
  const RowSum ps = walk.p, qs = walk.q;
  if (to2 == 0.0) {
    if (lead && tid == 0)
      p.next[b] = ps.first;
    return;
  }
  const bool residual = drawn && tried;
  const E* const prow = logits(0, row);
  const E* const qrow = logits(1, row);
  auto mark = [&](int piece) { // the tried tokens of a piece
    if (!tried || drawn)
      return;
    for (int i = tid; i < PIECE / 32; i += THREADS)
      gone[i] = 0;
    __syncthreads();
    for (int c = at + 1 + tid; c < (parents ? n : min(at + 2, n)); c += THREADS) {
      const int64_t x = parent(c) == at ? tokens[c] : -1;
      if (x >= 0 && x < p.V && x / PIECE == piece)
        atomicOr(&gone[x % PIECE / 32], 1u << (x % 32));
    }
    __syncthreads();
  };
  // What is left of a vector of 16 bytes of the last row: p without the tokens that were tried, or max(p - q, 0).  all: p.
  const double pn = 1.0 / ps.sum, qn = 1.0 / qs.sum;
  const bool fits = ManyWeights::fits(ps.top, to2) && (!residual || ManyWeights::fits(qs.top, to2)); // (uniform)
  const ManyWeights mp(table, ps.top, to2), mq(table, qs.top, to2);
  const double pm = fits ? pn * mp.off(ps.top) : 0.0, qm = fits && residual ? qn * mq.off(qs.top) : 0.0;
  struct Vector {
    uint4 p, q;
  };
  auto ask = [&](int piece, int i) { // vector i of a piece, where there is one
    const int from = piece * PIECE + i * N;
    return i < VECTORS ? Vector{load_raw<E>(prow, from, p.V), residual ? load_raw<E>(qrow, from, p.V) : uint4{}} : Vector{};
  };
  auto rest = [&](const Vector& v, int piece, int i, bool all, double (&w)[N]) {
    const int from = piece * PIECE + i * N;
    float x[N], y[N];
    raw_logits<E>(v.p, x);
    raw_logits<E>(v.q, y);
    const bool without = tried && !drawn && !all;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const float a = x[e] == x[e] ? x[e] : -INFINITY, z = y[e] == y[e] ? y[e] : -INFINITY;
      w[e] = fits ? mp(a) * pm : weight_of(a, ps.top, to2) * pn;
      if (residual && !all)
        w[e] = fmax(w[e] - (fits ? mq(z) * qm : weight_of(z, qs.top, to2) * qn), 0.0);
      if (without && gone[(from + e) % PIECE / 32] >> ((from + e) % 32) & 1)
        w[e] = 0.0;
      w[e] = from + e < p.V ? w[e] : 0.0;
    }
  };
  auto mine = [&](const Vector& v, int piece, int i, bool all, double (&w)[N]) { // and their sum
    double s = 0.0;
    if (i < VECTORS) {
      rest(v, piece, i, all, w);
#pragma unroll
      for (int e = 0; e < N; e++)
        s += w[e];
    }
    return s;
  };
  auto sum_of_piece = [&](int piece) { // in all threads; `gone` marked
    Vector v[EACH];
    double s = 0.0;
#pragma unroll
    for (int h = 0; h < EACH; h++)
      v[h] = ask(piece, h * THREADS + tid);
#pragma unroll
    for (int h = 0; h < EACH; h++) {
      double w[N];
      s += mine(v[h], piece, h * THREADS + tid, false, w);
    }
    s = reduce_lanes<64>(s, add64);
    __syncthreads();
    if (lane == 0)
      red[wave] = s;
    __syncthreads();
    double whole = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; i++)
      whole += red[i];
    return whole;
  };
  double* const sums = p.sums + (int64_t)b * p.C;
  if constexpr (DRAFTS) {
    if (residual) {
      const double s = sum_of_piece((int)blockIdx.y);
      if (tid == 0) { // (written through to the level that all XCDs share, and there before it counts)
        __hip_atomic_store(&sums[blockIdx.y], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        ended_last = __hip_atomic_fetch_add(&p.ended[b], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)p.C - 1;
      }
      __syncthreads();
      if (!ended_last)
        return;
    } else if (blockIdx.y) {
      return;
    }
  }
  auto sum_at = [&](int i) { return DRAFTS ? __hip_atomic_load(&sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : sums[i]; };
  {
    // The pieces' sums: from the first launch less the tried tokens' shares (a difference of sums near 1, so a rest that small is
    // summed anew, as it is where more were tried than are kept), from the second one, or, where nothing is left, p.
    bool all = !tried;
    for (int round = 0;; round++) {
      if (wave == 0) {
        auto of_piece = [&](int i) {
          if (i >= p.C)
            return 0.0;
          if (!all && (drawn || round > 0))
            return sum_at(i);
          const Piece z = load_piece<SHARED>(p.pieces + (int64_t)row * p.C + i);
          double s = z.sum > 0.0 ? z.sum * weight_of(z.top, ps.top, to2) * pn : 0.0;
          if (!all)
#pragma unroll 8
            for (int c = 0; c < min(tried, DRAFT_NODES); c++)
              s -= tried_in[c] == i ? tried_px[c] : 0.0;
          return fmax(s, 0.0);
        };
        const double head = of_piece(lane);
        const double head_run = scan64(head);
        double whole = __shfl(head_run, 63);
        for (int i0 = 64; i0 < p.C; i0 += 64)
          whole += reduce_lanes<64>(of_piece(i0 + lane), add64);
        const double border = (double)sample * whole;
        double before = 0.0, start = 0.0;
        int piece = -1, last = 0;
        for (int i0 = 0; i0 < p.C && piece < 0; i0 += 64) {
          const double s = i0 ? of_piece(i0 + lane) : head, run = i0 ? scan64(s) : head_run;
          const uint64_t beyond = __builtin_amdgcn_ballot_w64(s > 0.0 && before + run > border);
          const uint64_t some = __builtin_amdgcn_ballot_w64(s > 0.0);
          if (beyond) {
            piece = i0 + __builtin_ctzll(beyond);
            start = before + __shfl(run - s, __builtin_ctzll(beyond));
          } else if (some) { // (where the border is rounded past the last one)
            last = i0 + 63 - __builtin_clzll(some);
            start = before + __shfl(run - s, 63 - __builtin_clzll(some));
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
      if (fine || all)
        break;
      if (drawn || round > 0) {
        all = true;
        continue;
      }
      for (int i = 0; i < p.C; i++) { // too little for differences
        mark(i);
        const double s = sum_of_piece(i);
        if (tid == 0)
          sums[i] = s;
      }
      __syncthreads();
    }
    const int piece = piece_at;
    const double border = piece_border;
    Vector own[EACH]; // (one after the other in order)
    double w[EACH][N], s = 0.0;
#pragma unroll
    for (int h = 0; h < EACH; h++)
      own[h] = ask(piece, tid * EACH + h);
    mark(piece);
#pragma unroll
    for (int h = 0; h < EACH; h++)
      s += mine(own[h], piece, tid * EACH + h, all, w[h]);
    const double run = scan64(s);
    if (lane == 63)
      red[wave] = run;
    __syncthreads();
    double before = piece_before;
#pragma unroll
    for (int i = 0; i < WAVES - 1; i++)
      before += i < wave ? red[i] : 0.0;
    before += run - s;
    int found = p.V, last = -1;
    if (tid * EACH < VECTORS) {
#pragma unroll
      for (int h = 0; h < EACH; h++)
#pragma unroll
        for (int e = 0; e < N; e++) {
          before += w[h][e];
          const int x = piece * PIECE + (tid * EACH + h) * N + e;
          if (w[h][e] > 0.0) {
            last = x;
            found = before > border && found == p.V ? x : found;
          }
        }
    }
    // the first lane and the first wave that found one; a border that is rounded past the piece's last token: that one
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(found < p.V), some = __builtin_amdgcn_ballot_w64(last >= 0);
    if (lane == 0) {
      found_at[wave] = p.V;
      last_at[wave] = -1;
    }
    if (lanes && lane == __builtin_ctzll(lanes))
      found_at[wave] = found;
    if (some && lane == 63 - __builtin_clzll(some))
      last_at[wave] = last;
    __syncthreads();
    if (wave == 0) {
      const int f = found_at[min(lane, WAVES - 1)], z = last_at[min(lane, WAVES - 1)];
      const uint64_t first_wave = __builtin_amdgcn_ballot_w64(f < p.V), last_wave = __builtin_amdgcn_ballot_w64(z >= 0 && lane < WAVES);
      if (first_wave) {
        if (lane == __builtin_ctzll(first_wave))
          p.next[b] = f;
      } else if (last_wave) {
        if (lane == 63 - __builtin_clzll(last_wave))
          p.next[b] = z;
      } else if (lane == 0) {
        p.next[b] = 0;
      }
    }
  }
}

template <typename E, int NV, bool DRAFTS>
__global__ void __launch_bounds__(walk_threads(DRAFTS), 4)
draft_walk_kernel(const DraftsParams p) {
  walk_sequence<E, NV, DRAFTS, walk_threads(DRAFTS), false>(p, (int)blockIdx.x);
}

// Both in one launch, for up to 64 sequences: a piece counts for each sequence that has its row (so that every count is full in the end,
// whatever the bounds hold), and the workgroup that completes one goes on with it; nobody waits.
template <typename E>
__global__ void __launch_bounds__(DRAFT_THREADS)
draft_small_kernel(const DraftsParams p) {
  __shared__ uint64_t complete;
  const int tid = threadIdx.x, row = (int)blockIdx.x, piece = (int)blockIdx.y;
  int first = 0, n = 0;
  const bool some = (tid & 63) < p.B;
  if (some)
    bounds_of(p, tid & 63, first, n);
  const uint64_t mine = __builtin_amdgcn_ballot_w64(some && row >= first && row < first + n);
  const Piece r = piece_of_row<E, 1>(p, mine ? __builtin_ctzll(mine) : 0, row, piece, 0);
  if (tid < 64) {
    if (row == 0 && piece == 0 && some && n < 1) {
      p.count[tid] = 0;
      p.next[tid] = 0;
    }
    if (tid == 0) { // (there before it counts)
      uint64_t* const to = reinterpret_cast<uint64_t*>(p.pieces + (int64_t)row * p.C + piece);
      __hip_atomic_store(to, __builtin_bit_cast(uint64_t, r.sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(to + 1, (uint64_t)__float_as_uint(r.top) | (uint64_t)(uint32_t)r.first << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    bool last = false;
    if (mine >> tid & 1) {
      const unsigned most = (unsigned)(n * p.C) - 1;
      last = atomicInc(p.left + tid * DRAFT_STRIDE, most) == most;
    }
    const uint64_t done = __builtin_amdgcn_ballot_w64(last);
    if (tid == 0)
      complete = done;
  }
  __syncthreads();
  for (uint64_t todo = complete; todo; todo &= todo - 1) {
    walk_sequence<E, 1, false, DRAFT_THREADS, true>(p, __builtin_ctzll(todo));
    __syncthreads();
  }
}

static int64_t draft_pieces(int64_t V, int64_t size, int nv) { return (V * size + DRAFT_THREADS * 16 * nv - 1) / (DRAFT_THREADS * 16 * nv); }
// Vectors of 16 bytes that a thread takes of a row: four, which halves the instructions around the sums, or one where that leaves most of the
// CUs idle (5 rows of 32000 3.0 us, with four 4.0; 24 rows of 152000 7.1 + 10.6 for the walk, with four 5.3 + 9.6).
static int draft_vectors(int64_t rows, int64_t V, int64_t size) {
  return rows * draft_pieces(V, size, 4) >= 128 ? 4 : 1;
}

} // namespace tppx

using namespace tppx;

extern "C" int tppx_verify_drafts(const void* tokens, const void* target, const void* draft, int dtype, const void* cu, const void* parents,
                                  const void* uniforms, const void* sample, const void* temperatures, float temperature, void* path,
                                  void* count, void* next, int64_t T, int64_t B, int64_t V, int64_t t_ld, int64_t d_ld, void* ws,
                                  int64_t ws_bytes, void* counters, int64_t counter_bytes, tppx_stream_t stream) {
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
  TPPX_REQUIRE(ws_bytes >= 0 && (ws_bytes == 0 || ws) && counter_bytes >= 0 && (counter_bytes == 0 || counters), TPPX_EINVAL, "%s: size given with a null pointer", who);
  TPPX_REQUIRE(((uintptr_t)counters & 3u) == 0, TPPX_EINVAL, "%s: counters not 4-byte aligned", who);
  DraftsParams p;
  memset(&p, 0, sizeof(p));
  p.tokens = (const int64_t*)tokens; p.target = target; p.draft = draft; p.cu = (const int32_t*)cu; p.parents = (const int32_t*)parents;
  p.uniforms = (const float*)uniforms; p.sample = (const float*)sample; p.temps = (const float*)temperatures; p.to2 = temperature > 0.f ? LOG2E_64 / (double)temperature : 0.0;
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
  p.ended = (unsigned int*)(p.sums + (B * p.C + 1) / 2 * 2);
  p.rows = (RowSum*)(p.ended + (B + 3) / 4 * 4);
  p.nodes = (NodeShare*)(p.rows + 2 * T);
  // One launch: few rows, whose pieces 16 lanes look over in a few trips (5 rows of 32000 greedy 7.0 us, two launches 3.2 + 3.2, and with the
  // call from a program 13.3 and 15.6).
  p.left = nv == 1 && !draft && T > 0 && T <= 32 && B <= 64 && p.C <= 32 && B * DRAFT_STRIDE * 4 <= counter_bytes ? (unsigned int*)counters : nullptr;
  auto go = [&](auto e, auto nv_) {
    using E = decltype(e);
    constexpr int NV = decltype(nv_)::value;
    if (p.left) {
      draft_small_kernel<E><<<dim3((unsigned)T, (unsigned)p.C), dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
      return;
    }
    if (T > 0)
      draft_rows_kernel<E, NV><<<dim3((unsigned)T, (unsigned)p.C, (unsigned)p.sides), dim3(DRAFT_THREADS), 0, (hipStream_t)stream>>>(p);
    if (draft)
      draft_walk_kernel<E, NV, true><<<dim3((unsigned)B, (unsigned)p.C), dim3(walk_threads(true)), 0, (hipStream_t)stream>>>(p);
    else
      draft_walk_kernel<E, NV, false><<<dim3((unsigned)B), dim3(walk_threads(false)), 0, (hipStream_t)stream>>>(p);
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
  return (drafts ? 2 : 1) * T * C * (int64_t)sizeof(Piece) + (B * C + 1) / 2 * 16 + (B + 3) / 4 * 16 + T * (int64_t)(2 * sizeof(RowSum) + sizeof(NodeShare)) + 256;
}
