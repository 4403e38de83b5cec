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
