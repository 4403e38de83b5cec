// What the kernels of the MXFP4 cache and of packed prompts share.
#pragma once
#include <hip/hip_runtime.h>

#include "tppx_common.h"
#include "tppx_launch.h"
#include "tppx_norm.h"

namespace tppx {

// ---------------------------------------------------------------------------
// shared by the kernels
// ---------------------------------------------------------------------------
// sequence of a packed token: the number of sequences that end at or before it (64 ends per step, all lanes)
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int tok) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int i0 = 1; i0 <= B; i0 += 64)
    b += __popcll(__builtin_amdgcn_ballot_w64(i0 + lane <= B && cu[min(i0 + lane, B)] <= tok));
  return __builtin_amdgcn_readfirstlane(b);
}

// Workgroup `blk` of a launch whose sequences take ceil(tokens * per / rows) workgroups each: its sequence, that one's first
// row and tokens, and the workgroup's number inside it.  False past the last one.  All lanes of a wave take part.
// order(blk, all): the place of workgroup blk of `all`, applied for up to 64 sequences.
struct Block {
  int b, start, n, at;
};
template <typename F>
__device__ __forceinline__ bool locate(const int32_t* cu, int B, int T, int per, int rows, int blk, Block& o, F&& order) {
  if (!cu) { // one token per sequence
    const int each = (per + rows - 1) / rows;
    o.b = blk / each;
    o.at = blk - o.b * each;
    o.start = o.b;
    o.n = 1;
    return o.b < B;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int i0 = 0; i0 < B; i0 += 64) {
    const int i = min(i0 + lane, B - 1);
    const int s = min(max(cu[i], 0), T), e = min(max(cu[i + 1], 0), T);
    const int n = i0 + lane < B ? max(e - s, 0) : 0;
    const int c = (int)(((int64_t)n * per + rows - 1) / rows);
    int sum = c;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int t = __shfl_up(sum, d);
      sum += lane >= d ? t : 0;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (B <= 64)
      blk = order(blk, total);
    if (blk < before + total) {
      const int j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > blk));
      o.b = i0 + j;
      o.start = __builtin_amdgcn_readlane(s, j);
      o.n = __builtin_amdgcn_readlane(n, j);
      o.at = blk - before - (__builtin_amdgcn_readlane(sum, j) - __builtin_amdgcn_readlane(c, j));
      return true;
    }
    before += total;
  }
  return false;
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(f32x2_to_bf16_bits(f[0], f[1]), f32x2_to_bf16_bits(f[2], f[3]), f32x2_to_bf16_bits(f[4], f[5]),
                    f32x2_to_bf16_bits(f[6], f[7]));
}

__device__ __forceinline__ bool locate(const int32_t* cu, int B, int T, int per, int rows, int blk, Block& o) {
  return locate(cu, B, T, per, rows, blk, o, [](int b, int) { return b; });
}

// ---------------------------------------------------------------------------
// per-head norm and rotation: G lanes take a head's row, 16 channels each in two chunks of 8
// ---------------------------------------------------------------------------
template <int CTRL, typename A>
__device__ __forceinline__ A dpp_t(A v) {
  if constexpr (std::is_same_v<A, double>) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true), lo);
  } else {
    return dpp_mov<CTRL>(v);
  }
}
// sum over G adjacent lanes, in all of them
template <int G, typename A>
__device__ __forceinline__ A sum_of_lanes(A v) {
  v += dpp_t<0xB1>(v); // quad_perm [1,0,3,2]
  v += dpp_t<0x4E>(v); // quad_perm [2,3,0,1]
  if constexpr (G >= 8)
    v += dpp_t<0x141>(v); // row_half_mirror
  if constexpr (G >= 16)
    v += dpp_t<0x140>(v); // row_mirror
  return v;
}
__device__ __forceinline__ float rsqrt_t(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double rsqrt_t(double v) { // the hardware's estimate and two steps of Newton's method
  double r = __builtin_amdgcn_rsq(v);
  const double a = r * (1.5 - 0.5 * v * r * r);
  return v == (double)INFINITY ? r : a * (1.5 - 0.5 * v * a * a); // (of infinity zero, which Newton's step makes NaN)
}

// What the lanes of a row share out: chunks c[0], c[1] of 8 channels; their angles where they are rotated (adjacent pairs: four
// of each chunk, otherwise eight that both share).
struct Mx4Lane {
  int c[2];
  bool live, turn;
  float cs[8], sn[8];
};
template <int G, typename P>
__device__ __forceinline__ void mx4_share(const P& p, int u, Mx4Lane& t) {
  const int half = p.HR >> 4, rest = (p.H - p.HR) >> 4; // lanes of rotated chunks, of the others
  t.live = u < half + rest;
  t.c[0] = !t.live ? 0 : u < half ? u : u + half;
  t.c[1] = !t.live ? 0 : u < half ? u + half : u + half + rest;
}
// the angles of position `at` (outside the table: not rotated) for lane u
template <typename P>
__device__ __forceinline__ void mx4_angles(const P& p, int u, int64_t at, Mx4Lane& t) {
  t.turn = p.emb && at >= 0 && at < p.MP && u < (p.HR >> 4);
  if (t.turn) {
    const float* const c = p.emb + at * p.HR + (p.gptj ? p.HR >> 1 : 0);
    const float* const s = p.emb + (p.gptj ? at : p.MP + at) * p.HR;
    const int a0 = p.gptj ? t.c[0] * 4 : u * 8, a1 = p.gptj ? t.c[1] * 4 : u * 8 + 4;
    const f32x4 c0 = *reinterpret_cast<const f32x4*>(c + a0), c1 = *reinterpret_cast<const f32x4*>(c + a1);
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(s + a0), s1 = *reinterpret_cast<const f32x4*>(s + a1);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      t.cs[e] = c0[e];
      t.cs[4 + e] = c1[e];
      t.sn[e] = s0[e];
      t.sn[4 + e] = s1[e];
    }
  }
}

// a lane's 16 channels, normalised and rotated; all G lanes of the row take part
template <int G, typename A, typename P>
__device__ __forceinline__ void mx4_turn(const P& p, const uint4 (&w)[2], const Mx4Lane& t, const void* gamma, A (&y)[2][8]) {
#pragma unroll
  for (int h = 0; h < 2; h++) {
    float f[8];
    unpack8(w[h], f);
#pragma unroll
    for (int e = 0; e < 8; e++)
      y[h][e] = f[e];
  }
  if (gamma) {
    A ss = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 8; e++)
        ss = fma(y[h][e], y[h][e], ss);
    ss = sum_of_lanes<G>(ss);
    const A r = rsqrt_t(ss * ((A)1 / (A)p.H) + (A)p.eps);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float g[8];
      if (p.gamma_f32) {
        const f32x4* s = reinterpret_cast<const f32x4*>(gamma) + t.c[h] * 2;
        const f32x4 a = s[0], b = s[1];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          g[e] = a[e];
          g[4 + e] = b[e];
        }
      } else {
        unpack8(reinterpret_cast<const uint4*>(gamma)[t.c[h]], g);
      }
#pragma unroll
      for (int e = 0; e < 8; e++)
        y[h][e] = y[h][e] * r * (A)g[e];
    }
  }
  if (!t.turn)
    return;
  auto rotate = [&](A& a, A& b, float c, float s) {
    const A x = a, z = b;
    if constexpr (std::is_same_v<A, float>) {
      a = rotate_first(x, z, c, s);
      b = rotate_second(x, z, c, s);
    } else {
      asm("" : "+v"(c), "+v"(s)); // (not as 32 registers of fp64 over the whole loop)
      a = x * (A)c - z * (A)s;
      b = z * (A)c + x * (A)s;
    }
  };
  if (p.gptj) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        rotate(y[h][2 * e], y[h][2 * e + 1], t.cs[4 * h + e], t.sn[4 * h + e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      rotate(y[0][e], y[1][e], t.cs[e], t.sn[e]);
  }
}

// eight E2M1 codes of a dword times the scale, exact in bf16
__device__ __forceinline__ bf16x8 mx4_to_bf16(uint32_t codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

struct Mx4AttnParams {
  const uint16_t* q; // [T][Nq][H], rows q_ld elements apart
  const uint16_t *k, *v; // packed prompts: [T][Nkv][H], rows k_ld, v_ld elements apart
  int64_t q_ld, k_ld, v_ld;
  const uint8_t *kq, *ks, *vq, *vs;
  const int32_t *past, *cu;
  const uint16_t* mask; // [B][mask_ld], added to the scores, or null
  uint16_t* out;        // [T][Nq][H] contiguous
  float* part;          // [workgroup x][split][cols][H], then [workgroup x][split][cols][2]
  unsigned int* counters;
  int T, B, Nq, Nkv, R, Smax, mask_ld, splits, cols;
  float scale;
};
constexpr int MX4_COUNTER_STRIDE = 64; // arrival counters are 256 bytes apart

// The number of keys before a sequence's tokens, so that its sums with numbers of tokens and of keys (both below 2^30) stay in 32
// bits: more than the cache holds is all of it, and what lies 2^30 before the first slot sees none of it.
__device__ __forceinline__ int mx4_past(int past, int Smax) { return min(max(past, -(1 << 30)), Smax); }

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x3 __attribute__((ext_vector_type(3)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// maximum over the four 16-lane groups
__device__ __forceinline__ float max_of_groups(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ bool mx4_non_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}
// the pair with what is not finite set to zero
__device__ __forceinline__ uint32_t mx4_finite(uint32_t pair) {
  return ((pair & 0x7f80u) == 0x7f80u ? 0u : pair & 0xffffu) | ((pair & 0x7f800000u) == 0x7f800000u ? 0u : pair & 0xffff0000u);
}

// ---------------------------------------------------------------------------
// bf16 rows of keys and values in LDS, brought by loads straight into it: the chunks of 16 bytes of a row lie permuted (those loads
// write 1024 bytes in a row), so that neither the rows of a K operand nor the pieces that the transposing read of V takes meet in a bank
// ---------------------------------------------------------------------------
constexpr int packed_k_turn(int NJ, int row) { return NJ % 4 == 0 ? row & 15 : NJ % 2 == 0 ? (row >> 1) & 7 : (row >> 2) & 3; }
constexpr int packed_v_turn(int NJ, int row) { return 2 * (NJ % 4 == 0 ? row & 7 : NJ % 2 == 0 ? (row >> 1) & 3 : (row >> 2) & 1); }

// The transposing reads of V for 32 keys and N pieces of 16 channels, issued and waited for in one block (around the builtin the
// compiler waits for every load into LDS under way): piece d at a[d % X] + d / X * STEP, keys 16 .. 31 at + ROWS.
template <int OFF, int ROWS>
__device__ __forceinline__ void packed_v_operands(i32x2 (&v)[8][2], const uint32_t (&a)[8]) {
  asm volatile("ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %1, %16 offset:%25\n\t"
               "ds_read_b64_tr_b16 %2, %17 offset:%24\n\tds_read_b64_tr_b16 %3, %17 offset:%25\n\t"
               "ds_read_b64_tr_b16 %4, %18 offset:%24\n\tds_read_b64_tr_b16 %5, %18 offset:%25\n\t"
               "ds_read_b64_tr_b16 %6, %19 offset:%24\n\tds_read_b64_tr_b16 %7, %19 offset:%25\n\t"
               "ds_read_b64_tr_b16 %8, %20 offset:%24\n\tds_read_b64_tr_b16 %9, %20 offset:%25\n\t"
               "ds_read_b64_tr_b16 %10, %21 offset:%24\n\tds_read_b64_tr_b16 %11, %21 offset:%25\n\t"
               "ds_read_b64_tr_b16 %12, %22 offset:%24\n\tds_read_b64_tr_b16 %13, %22 offset:%25\n\t"
               "ds_read_b64_tr_b16 %14, %23 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]),
                 "=&v"(v[3][1]), "=&v"(v[4][0]), "=&v"(v[4][1]), "=&v"(v[5][0]), "=&v"(v[5][1]), "=&v"(v[6][0]), "=&v"(v[6][1]),
                 "=&v"(v[7][0]), "=&v"(v[7][1])
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "n"(OFF), "n"(OFF + ROWS)
               : "memory");
}
template <int OFF, int ROWS>
__device__ __forceinline__ void packed_v_operands(i32x2 (&v)[4][2], const uint32_t (&a)[4]) {
  asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
               "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
               "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
               "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]),
                 "=&v"(v[3][1])
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF), "n"(OFF + ROWS)
               : "memory");
}
template <int OFF, int ROWS> // (96 wide: six pieces at two addresses)
__device__ __forceinline__ void packed_v_operands(i32x2 (&v)[6][2], const uint32_t (&a)[2]) {
  asm volatile("ds_read_b64_tr_b16 %0, %12 offset:%14\n\tds_read_b64_tr_b16 %1, %12 offset:%15\n\t"
               "ds_read_b64_tr_b16 %2, %13 offset:%14\n\tds_read_b64_tr_b16 %3, %13 offset:%15\n\t"
               "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %12 offset:%17\n\t"
               "ds_read_b64_tr_b16 %6, %13 offset:%16\n\tds_read_b64_tr_b16 %7, %13 offset:%17\n\t"
               "ds_read_b64_tr_b16 %8, %12 offset:%18\n\tds_read_b64_tr_b16 %9, %12 offset:%19\n\t"
               "ds_read_b64_tr_b16 %10, %13 offset:%18\n\tds_read_b64_tr_b16 %11, %13 offset:%19\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]),
                 "=&v"(v[3][1]), "=&v"(v[4][0]), "=&v"(v[4][1]), "=&v"(v[5][0]), "=&v"(v[5][1])
               : "v"(a[0]), "v"(a[1]), "n"(OFF), "n"(OFF + ROWS), "n"(OFF + 64), "n"(OFF + 64 + ROWS), "n"(OFF + 128), "n"(OFF + 128 + ROWS)
               : "memory");
}

// 16 bytes per lane straight into LDS, 1024 in a row from `to` on
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t src, uint8_t* to, uint32_t offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)to, 16, offset, 0, 0, 0);
}

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LOWEST = -3.4028234e38f; // below every finite score, the bf16 lowest of a mask among them

// f(head size / 32) for the head sizes that are built
template <typename F>
inline void mx4_for_head(int H, F&& f) {
  switch (H) {
    case 64: f(std::integral_constant<int, 2>{}); break;
    case 96: f(std::integral_constant<int, 3>{}); break;
    case 128: f(std::integral_constant<int, 4>{}); break;
    case 192: f(std::integral_constant<int, 6>{}); break;
    default: f(std::integral_constant<int, 8>{});
  }
}
inline bool mx4_has_head(int64_t H) { return H == 64 || H == 96 || H == 128 || H == 192 || H == 256; }

int mx4_prompt_launch(const char* who, const Mx4AttnParams& p, int H, bool cache, hipStream_t stream);

} // namespace tppx
