// Key/value cache in MXFP4 (E2M1 codes, one E8M0 scale per 32 channels of a head) for sequences of different lengths, and
// attention of packed prompts: per-head norms with the rotation and the append, single and few tokens over the cache with
// the keys split over workgroups, and causal attention of prompts over packed bf16 rows or over the cache.
//
// Cache of a layer: codes [B][Nkv][Smax][H/2] (channel 2i of a byte in its low half), scales [B][Nkv][Smax][H/32], for the
// keys and for the values.  Tokens are packed: sequence b owns rows cu[b] .. cu[b + 1] - 1 of q, k, v and out, and held past[b]
// keys before them; cu null: one token per sequence.  Both arrays live on the device and are clamped there, so that no value in
// them leads out of a buffer.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "tppx_mx4.h"

namespace tppx {

// ---------------------------------------------------------------------------
// Norm, rotation and append.  G lanes take a head's row, 16 channels each in two chunks of 8: chunk l and the one it is rotated with,
// so that no channel changes lanes; behind the rotated ones chunk l and one half of the rest away.  The mean square is a sum over
// the G lanes.
//   y = x * (1 / sqrt(mean(x^2) + eps)) * gamma;  y' = y cos -+ partner sin
// A query is computed in fp32 and rounded once, to bf16.  A key that goes to the cache is computed in fp64: its code is a step
// function of the value, and in fp32 one in some 10^6 falls on the other side of a border than the formula's.  Codes: scale
// 2^(floor(log2 max) - 2), nearest, ties to the even code, 6 at most, as the MXFP4 weights; a block whose maximum is below 2^-124 is
// zero, one that holds an infinity or a NaN has scale byte 255 and reads back as NaN.  A block is four chunks: those of four
// adjacent lanes (ALIGNED: rotated width and rest are multiples of 64), or found chunk by chunk.
// What bounds it: the bytes, from some hundred tokens on (2027 tokens of 32 + 2 x 32 heads of 128 into the cache 110 MB in 21 us, 5.2 TB/s,
// the rate of a large copy; 2048 of 32 + 8 without it 78 MB in 14.3 us, 5.4 TB/s).  One token: the launch and one way to memory and back,
// 2.9 us, 3.8 with the append.
// ---------------------------------------------------------------------------
struct Mx4RowsParams {
  const uint16_t *q, *k, *v; // [T][heads][H], rows q_ld, k_ld, v_ld elements apart; q or v may be null
  uint16_t *qo, *ko, *vo;    // [T][heads][H] contiguous; with the cache ko, vo may be null (the values that the codes stand for)
  uint8_t *kq, *ks, *vq, *vs;
  const void *gq, *gk;       // [H] f32 or bf16, or null
  const float* emb;          // [2][MP][HR] cos / sin, or with gptj [MP][HR] sin | cos, or null
  const int64_t* pos;        // [T], or null: the slot in the cache
  const int32_t *past, *cu;
  int64_t q_ld, k_ld, v_ld;
  int T, B, Nq, Nkv, H, MP, HR, Smax;
  int gptj, gamma_f32;
  float eps;
};

// biased fp32 exponent (up to 2047 from fp64, kept in that bias) of the largest magnitude of 8 values
template <typename A>
__device__ __forceinline__ int top_exponent(const A (&y)[8]) {
  int top = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    if constexpr (std::is_same_v<A, double>)
      top = max(top, (__double2hiint(y[e]) >> 20) & 0x7ff);
    else
      top = max(top, (int)((__float_as_uint(y[e]) >> 23) & 0xffu));
  }
  return top;
}
// codes of 8 values of a block with that scale byte (a dword).  The conversion is the hardware's, nearest even and 6 at most; it
// keeps the sign of a zero, which is dropped.  A fp64 value enters as fp32 by its upper dword, with the last bit set where the lower
// one is not zero: every border between two codes has both zero, so that it stays on its side of all of them.  The division by the
// scale is a difference of exponents there; what is below 2^-15 of it becomes 2^-15, whose code is zero too.
template <typename A>
__device__ __forceinline__ uint32_t mx4_encode(const A (&y)[8], int byte) {
  if (byte == 0 || byte == 255)
    return 0;
  uint32_t q = 0;
  if constexpr (std::is_same_v<A, double>) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t hi = (uint32_t)__double2hiint(y[e]) | (__double2loint(y[e]) != 0 ? 1u : 0u);
      const int t = max((int)(hi & 0x7fffffffu) + (127 - byte) * (1 << 20), 0x3f000000);
      f[e] = __uint_as_float((((uint32_t)t << 3) - (896u << 23)) | (hi & 0x80000000u));
    }
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[0], f[1], 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[2], f[3], 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[4], f[5], 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[6], f[7], 1.0f, 3);
  } else {
    const float s = e8m0_to_f32((uint32_t)byte);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[0], y[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[2], y[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[4], y[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[6], y[7], s, 3);
  }
  const uint32_t nz = (q | (q >> 1) | (q >> 2)) & 0x11111111u;
  return q & (0x77777777u | (nz << 3));
}

template <int G, bool CACHE, bool ALIGNED>
__global__ void __launch_bounds__(256, ALIGNED ? CACHE ? 4 : 5 : 3)
mx4_rows_kernel(const Mx4RowsParams p) {
  // A thread's token stays, the heads go by: a wave works on one head (of q, k or v) of 64 / G tokens in a row, whose rows in
  // the cache lie side by side, and a token's angles are read once.
  constexpr int TB = 256 / G; // tokens of a workgroup
  const int u = threadIdx.x % G, mine = (int)blockIdx.x * TB + (int)threadIdx.x / G, tok = min(mine, p.T - 1);
  const int nq = p.q ? p.Nq : 0, nk = p.Nkv, total = nq + nk + (p.v ? p.Nkv : 0);
  const int half = p.HR >> 4, rest = (p.H - p.HR) >> 4; // lanes of rotated chunks, of the others
  Mx4Lane t;
  mx4_share<G>(p, u, t);
  // rows of a token: queries, then keys, then values; the next one is under way while one is worked on
  uint4 next[2];
  auto load = [&](int i) {
    if (i >= total)
      return;
    const uint16_t* const src = i < nq ? p.q + (int64_t)i * p.H : i < nq + nk ? p.k + (int64_t)(i - nq) * p.H : p.v + (int64_t)(i - nq - nk) * p.H;
    const uint4* const at = reinterpret_cast<const uint4*>(src + (int64_t)tok * (i < nq ? p.q_ld : i < nq + nk ? p.k_ld : p.v_ld));
    next[0] = at[t.c[0]];
    next[1] = at[t.c[1]];
  };
  int row = (int)blockIdx.y;
  load(row);
  int b = 0;
  int64_t slot = 0; // (past may hold anything: in 64 bits)
  bool here = mine < p.T;
  if (CACHE) {
    int first = tok;
    b = tok;
    if (p.cu) {
      b = sequence_of(p.cu, p.B, __builtin_amdgcn_readfirstlane(tok)); // of the wave's first token
      while (b < p.B && p.cu[b + 1] <= tok)
        b++;
      here = here && b < p.B && tok >= p.cu[0]; // (not a row behind the last sequence)
      b = min(b, p.B - 1);
      first = p.cu[b];
    }
    slot = (int64_t)p.past[b] + tok - first;
  }
  const int64_t at = p.pos ? p.pos[tok] : slot;
  const bool room = slot >= 0 && slot < p.Smax;
  mx4_angles(p, u, at, t);
  uint4 w[2];
  auto step = [&]() {
    w[0] = next[0];
    w[1] = next[1];
    if (!t.live) // (heads of 96 and 192 leave lanes over)
      w[0] = w[1] = make_uint4(0, 0, 0, 0);
    load(row + (int)gridDim.y);
  };
  auto write = [&](uint16_t* to, int heads, int i, const float (&y)[2][8]) { // a row of [T][heads][H]
    if (!t.live || !here)
      return;
    uint4* const dst = reinterpret_cast<uint4*>(to + ((int64_t)tok * heads + i) * p.H);
    dst[t.c[0]] = pack8(y[0]);
    dst[t.c[1]] = pack8(y[1]);
  };
  auto append = [&](auto& y, uint8_t* codes_at, uint8_t* scales_at, uint16_t* held, int i) {
    using A = std::remove_reference_t<decltype(y[0][0])>;
    constexpr int TOP = std::is_same_v<A, double> ? 0x7ff : 0xff, BIAS = std::is_same_v<A, double> ? 1023 : 127;
    int top[2] = {top_exponent(y[0]), top_exponent(y[1])};
    if constexpr (ALIGNED) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        top[h] = max(top[h], __builtin_amdgcn_update_dpp(0, top[h], 0xB1, 0xf, 0xf, true));
        top[h] = max(top[h], __builtin_amdgcn_update_dpp(0, top[h], 0x4E, 0xf, 0xf, true));
      }
    } else {
      const int lane0 = (threadIdx.x & 63) & ~(G - 1), own[2] = {top[0], top[1]};
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int ch = (t.c[h] & ~3) + j, r = ch - 2 * half; // lane and slot that hold chunk ch
          const bool second = r < 0 ? ch >= half : r >= rest;
          const int src = lane0 + (r < 0 ? ch - (second ? half : 0) : half + r - (second ? rest : 0));
          const int a = __shfl(own[0], src), z = __shfl(own[1], src);
          top[h] = max(top[h], second ? z : a);
        }
    }
    const int64_t to = ((int64_t)b * p.Nkv + i) * p.Smax + slot;
    float f[2][8];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int byte = top[h] == TOP ? 255 : min(max(top[h] - BIAS + 125, 0), 254);
      const uint32_t codes = mx4_encode(y[h], byte);
      if (t.live && here && room) {
        *reinterpret_cast<uint32_t*>(codes_at + to * (p.H >> 1) + t.c[h] * 4) = codes;
        if ((t.c[h] & 3) == 0)
          scales_at[to * (p.H >> 5) + (t.c[h] >> 2)] = (uint8_t)byte;
      }
      if (held) {
        typedef __attribute__((ext_vector_type(2))) float f32x2;
        const float s = e8m0_to_f32((uint32_t)byte);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const f32x2 v = e == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0) : e == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1)
                        : e == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
          f[h][2 * e] = v[0] * s;
          f[h][2 * e + 1] = v[1] * s;
        }
      }
    }
    if (held)
      write(held, p.Nkv, i, f);
  };
  for (; row < nq; row += (int)gridDim.y) {
    step();
    float y[2][8];
    mx4_turn<G>(p, w, t, p.gq, y);
    write(p.qo, p.Nq, row, y);
  }
  for (; row < nq + nk; row += (int)gridDim.y) {
    step();
    if constexpr (CACHE) {
      double y[2][8];
      mx4_turn<G>(p, w, t, p.gk, y);
      append(y, p.kq, p.ks, p.ko, row - nq);
    } else {
      float y[2][8];
      mx4_turn<G>(p, w, t, p.gk, y);
      write(p.ko, p.Nkv, row - nq, y);
    }
  }
  if constexpr (CACHE)
    for (; row < total; row += (int)gridDim.y) {
      step();
      float y[2][8];
      unpack8(w[0], y[0]);
      unpack8(w[1], y[1]);
      append(y, p.vq, p.vs, p.vo, row - nq - nk);
    }
}

// ---------------------------------------------------------------------------
// Few tokens over the cache, keys split over workgroups.  The columns of a sequence's K/V head are its (token, query head)
// pairs; a workgroup takes 16 of them, the columns of a 16 x 16 x 32 MFMA, so that a cached row is read once for all of them
// and with one token per sequence and up to 16 heads per K/V head once in all.  Both products run transposed:
//   scores^T[key][col] = K Q^T,  out^T[channel][col] += V^T P^T,
// the score tile's register layout being the second operand's of the V product.
// A wave works by itself on tiles of 64 keys.  Keys: lane (g, c) holds channels g * H/4 .. of key c of a run of 16: whole blocks
// (or parts of one), 4 H/32 bytes of codes loaded where they lie, no LDS; the channels an MFMA step sums over are the same
// permutation for the query.  Values: a row's codes go to the wave's own LDS and come back by the transposing read for 4-bit
// elements: of 16 lanes, lane i fetches 16 channels (8 bytes) of key i and gets the 16 keys of channel i.
// A value's scale belongs to (key, block), in the transposed operand it differs from slot to slot, so it multiplies the
// probability instead: P is rounded to bf16 and the exponent of each block's scale is added to it as an integer (exact; what
// falls below bf16's range is zero), the codes enter unscaled.  A probability of zero stays zero whatever the scale, so a key that a
// column does not see adds nothing, also where its block is NaN; blocks of seen keys that are NaN (scale byte 255) are found
// by their bytes and put into the result.
// Scores, maximum and sums in fp32; the probabilities' sum is that of the bf16 ones, taken by an MFMA with ones.
// What bounds it: large layers the cache's bytes (32 sequences x 16000 keys x 8 K/V heads of 128, 558 MB: 88 us, 6.3 TB/s; a large
// copy moves 5.15, in and out); smaller ones a wave's way through a tile (about a microsecond: loads, two chains of matrix instructions, the
// softmax between them), the number of tiles that it takes one after the other, and the merge behind them (1 x 2048 keys of 32 heads,
// 8.9 MB: 7.0 us; 16 uneven sequences of 64 heads on 8, 20 MB: 14.0 .. 14.6).  The bf16 cache's kernel takes 85 us for 16 x 2048 keys of 32 heads, this
// one 25.
// ---------------------------------------------------------------------------
template <int NJ>
constexpr int mx4_scale_bytes() { // scale bytes of a lane's channels of a key: whole blocks, or one that they lie in
  return NJ % 4 == 0 ? NJ / 4 : NJ <= 2 ? 1 : NJ;
}

template <int NJ, int W, bool MASK, bool STREAM>
__global__ void __launch_bounds__(W * 64)
mx4_split_kernel(const Mx4AttnParams p) {
  constexpr int H = 32 * NJ, RB = 16 * NJ;          // bytes of a row's codes
  constexpr int PITCH = RB + 16;                     // of a row in LDS: 16 rows of a group on different banks
  constexpr int SD = NJ > 4 ? 2 : 1;                 // dwords of a row's scales in registers
  constexpr int WAVE_LDS = 64 * PITCH + 128 * NJ;    // per wave: codes of the rows, exponents [block][row]
  constexpr int OP = H + 4;                          // pitch of a merged output row in floats
  constexpr int MERGE = (W * 16 * OP + W * 32) * 4, LDS = W * WAVE_LDS > MERGE ? W * WAVE_LDS : MERGE;
  constexpr int NS = mx4_scale_bytes<NJ>();
  constexpr int AUX = STREAM ? 2 : 0; // codes with the non-temporal hint
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ float merged[16][33]; // weights of the splits, then the sum
  __shared__ int arrived_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int hk = (int)blockIdx.x % p.Nkv;
  Block o;
  if (!locate(p.cu, p.B, p.T, p.R, 16, (int)blockIdx.x / p.Nkv, o))
    return;
  const int ncol = min(16, o.n * p.R - o.at * 16); // of this workgroup
  const int col = o.at * 16 + min(c, ncol - 1), tok = col / p.R, r0 = col - tok * p.R;
  const int past = mx4_past(p.past[o.b], p.Smax);
  const int limit = min(max(past + tok + 1, 0), p.Smax); // keys this lane's column sees
  const int L = min(max(past + (o.at * 16 + ncol - 1) / p.R + 1, 0), p.Smax);
  const int S = max(min(p.splits, (L + W * 64 - 1) / (W * 64)), 1); // splits that have keys; the others take no part
  if ((int)blockIdx.y >= S)
    return;

  const int64_t head = ((int64_t)o.b * p.Nkv + hk) * p.Smax;
  const uint8_t* const kq = p.kq + head * RB;
  const uint8_t* const ks = p.ks + head * NJ;
  const uint8_t* const vq = p.vq + head * RB;
  const uint8_t* const vs = p.vs + head * NJ;
  const uint16_t* mrow = MASK ? p.mask + (int64_t)o.b * p.mask_ld : nullptr;

  bf16x8 q[NJ];
  {
    const uint16_t* qrow = p.q + (int64_t)(o.start + tok) * p.q_ld + (hk * p.R + r0) * H + g * (8 * NJ);
#pragma unroll
    for (int j = 0; j < NJ; j++)
      q[j] = *reinterpret_cast<const bf16x8*>(qrow + j * 8);
  }
  uint32_t kc[4][NJ], kb[4][NS]; // keys of the tile: codes and scale bytes
  i32x4 vc[NJ];                  // values: 16-byte chunks i * 64 + lane of the tile's rows
  uint32_t vb[SD];               // scales of the value of key `lane`
  // (buffers of the tile's rows: what lies past the cache's end reads as zero, with no branch and no access)
  auto rsrc = [](const uint8_t* at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at), 0, bytes, 0x00020000);
  };
  auto request_k = [&](int base) {
    const int rows = min(max(p.Smax - base, 0), 64);
    const auto codes = rsrc(kq + (int64_t)base * RB, rows * RB);
    const auto scales = rsrc(ks + (int64_t)base * NJ, rows * NJ);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int at = (t * 16 + c) * RB + g * (4 * NJ);
      if constexpr (NJ == 2 || NJ == 6) {
        const i32x2 w = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(codes, at, 0, AUX));
        kc[t][0] = (uint32_t)w[0];
        kc[t][1] = (uint32_t)w[1];
      } else if constexpr (NJ == 3) {
        const i32x3 w = __builtin_bit_cast(i32x3, __builtin_amdgcn_raw_buffer_load_b96(codes, at, 0, AUX));
        kc[t][0] = (uint32_t)w[0];
        kc[t][1] = (uint32_t)w[1];
        kc[t][2] = (uint32_t)w[2];
      }
#pragma unroll
      for (int j = NJ % 4 == 3 ? NJ : NJ % 4; j + 4 <= NJ; j += 4) {
        const i32x4 w = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, at + j * 4, 0, AUX));
#pragma unroll
        for (int d = 0; d < 4; d++)
          kc[t][j + d] = (uint32_t)w[d];
      }
#pragma unroll
      for (int j = 0; j < NS; j++)
        kb[t][j] = __builtin_amdgcn_raw_buffer_load_b8(scales, (t * 16 + c) * NJ + (NJ % 4 == 0 ? g * NS + j : (g * NJ + j) >> 2), 0, 0);
    }
  };
  auto request_v = [&](int base) {
    const int rows = min(max(p.Smax - base, 0), 64);
    const auto codes = rsrc(vq + (int64_t)base * RB, rows * RB);
    const auto scales = rsrc(vs + (int64_t)base * NJ, rows * NJ);
#pragma unroll
    for (int i = 0; i < NJ; i++)
      vc[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, (i * 64 + lane) * 16, 0, AUX));
    if constexpr (NJ == 4) {
      vb[0] = __builtin_amdgcn_raw_buffer_load_b32(scales, lane * 4, 0, 0);
    } else if constexpr (NJ == 8) {
      const i32x2 w = __builtin_bit_cast(i32x2, __builtin_amdgcn_raw_buffer_load_b64(scales, lane * 8, 0, 0));
      vb[0] = (uint32_t)w[0];
      vb[1] = (uint32_t)w[1];
    } else if constexpr (NJ == 2) {
      vb[0] = __builtin_amdgcn_raw_buffer_load_b16(scales, lane * 2, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < SD; j++)
        vb[j] = 0;
#pragma unroll
      for (int j = 0; j < NJ; j++)
        vb[j >> 2] |= (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(scales, lane * NJ + j, 0, 0) << (8 * (j & 3));
    }
  };

  uint8_t* const mine = lds + wave * WAVE_LDS;
  // key t * 16 + g * 4 + r of the tile lies at row g * 16 + t * 4 + r: the order in which lane group g holds its probabilities
  auto place = [](int key) { return ((key >> 2) & 3) * 16 + (key >> 4) * 4 + (key & 3); };
  float m = LOWEST;
  f32x4 acc[2 * NJ], sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int dt = 0; dt < 2 * NJ; dt++)
    acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
  const float to2 = MASK ? LOG2E : p.scale * LOG2E; // of a score in powers of two

  const int step = S * W * 64;
  int base = ((int)blockIdx.y * W + wave) * 64;
  if (base < L) {
    request_k(base);
    request_v(base);
  }
  for (; base < L; base += step) {
    f32x4 sc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        const uint32_t byte = kb[t][NJ % 4 == 0 ? j >> 2 : NS == 1 ? 0 : j];
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx4_to_bf16(kc[t][j], e8m0_to_f32(byte)), q[j], sc[t], 0, 0, 0);
      }
    }
    const bool more = base + step < L; // wave-uniform
    if (more)
      request_k(base + step);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; i++)
      x[i] = MASK ? sc[i >> 2][i & 3] * p.scale : sc[i >> 2][i & 3];
    if (MASK) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = base + (i >> 2) * 16 + g * 4 + (i & 3);
        const float mv = key < p.mask_ld ? bf16_bits_to_f32(mrow[min(key, p.mask_ld - 1)]) : 0.f;
        x[i] = mv == -INFINITY ? -INFINITY : x[i] + mv; // (a key that is not looked at may be NaN)
      }
    }
    if (base + 64 > min(past + 1, p.Smax)) { // wave-uniform: some column may not see some key
#pragma unroll
      for (int i = 0; i < 16; i++)
        x[i] = base + (i >> 2) * 16 + g * 4 + (i & 3) < limit ? x[i] : -INFINITY;
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < 16; i++)
      mx = fmaxf(mx, x[i]);
    // The maximum is followed at once: the largest probability is then exactly 1, and the relative error against 64 bits 1.8e-3 for
    // 16000 keys (2.3e-3 where it follows in steps of 2^8, which saves less than 1 % here).
    if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
      mx = max_of_groups(mx);
      const float alpha = __builtin_amdgcn_exp2f((m - mx) * to2);
#pragma unroll
      for (int dt = 0; dt < 2 * NJ; dt++)
        acc[dt] *= alpha;
      sum *= alpha;
      m = mx;
    }
    const float off = -m * to2;
    uint32_t pr[8]; // bf16 pairs, slots 2 e, 2 e + 1
#pragma unroll
    for (int e = 0; e < 8; e++) { // (with a mask the difference first: its lowest value times log2 e is no number)
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; h++)
        f[h] = __builtin_amdgcn_exp2f(MASK ? (x[2 * e + h] - m) * to2 : fmaf(x[2 * e + h], to2, off));
      pr[e] = f32x2_to_bf16_bits(f[0], f[1]);
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const i32x4 w = {(int)pr[4 * u], (int)pr[4 * u + 1], (int)pr[4 * u + 2], (int)pr[4 * u + 3]};
      sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, w), sum, 0, 0, 0);
    }
    // the values' codes and scales through LDS (the wave's own: its accesses to LDS stay in order)
    const bool odd = base + lane < L && [&] {
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < SD; j++)
        any |= ((vb[j] & 0x7f7f7f7fu) + 0x01010101u) & vb[j] & 0x80808080u;
      return any != 0;
    }();
#pragma unroll
    for (int i = 0; i < NJ; i++) {
      const int ch = i * 64 + lane;
      *reinterpret_cast<i32x4*>(mine + place(ch / NJ) * PITCH + (ch % NJ) * 16) = vc[i];
    }
    {
      // a scale as what it adds to the bits of a bf16; rows past the keys may hold anything: what makes every sum negative
      uint16_t* const dst = reinterpret_cast<uint16_t*>(mine + 64 * PITCH) + place(lane);
      const bool live = base + lane < L;
#pragma unroll
      for (int bl = 0; bl < NJ; bl++)
        dst[bl * 64] = (uint16_t)(live ? ((vb[bl >> 2] >> (8 * (bl & 3))) & 0xffu) * 128u - 127u * 128u : 0x8000u);
    }
    if (more)
      request_v(base + step);
    const i32x4* const exps = reinterpret_cast<const i32x4*>(mine + 64 * PITCH) + g * 2; // [block][8]: of this group's 16 rows
    if (__builtin_amdgcn_ballot_w64(odd) != 0) { // a block of NaN: into the columns that see its key
#pragma unroll
      for (int bl = 0; bl < NJ; bl++) {
        int bad = 0;
#pragma unroll
        for (int i = 0; i < 16; i++)
          bad |= reinterpret_cast<const uint16_t*>(exps + bl * 8)[i] == 128 * 128 && x[i] != -INFINITY;
        bad |= __shfl_xor(bad, 16);
        bad |= __shfl_xor(bad, 32);
        if (bad)
          acc[2 * bl] = acc[2 * bl + 1] = f32x4{NAN, NAN, NAN, NAN};
      }
    }
    // A probability of zero as the lowest integer, so that no scale lifts it; the sums saturate, negative ones are zero.
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint32_t some; // 1 where it is not zero (the compiler makes conditions of it)
      asm("v_pk_min_u16 %0, %1, %2" : "=v"(some) : "v"(pr[e]), "s"(0x00010001u));
      asm("v_pk_mad_u16 %0, %1, %2, %3" : "=v"(pr[e]) : "v"(some), "s"(0x80008000u), "v"(pr[e] ^ 0x80008000u));
    }
    const uint8_t* const vrow = mine + (g * 16 + c) * PITCH;
#pragma unroll
    for (int bl = 0; bl < NJ; bl++) {
      i32x4 w[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const i32x4 ex = exps[bl * 8 + h];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t t;
          asm("v_pk_add_i16 %0, %1, %2 clamp" : "=v"(t) : "v"(ex[e]), "v"(pr[h * 4 + e]));
          w[h][e] = __builtin_bit_cast(int, __builtin_elementwise_max(__builtin_bit_cast(i16x2, t), i16x2{0, 0}));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int dt = 2 * bl + h;
        const i32x2 codes = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2*)(vrow + dt * 8));
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx4_to_bf16((uint32_t)codes[0], 1.0f), __builtin_bit_cast(bf16x8, w[0]), acc[dt], 0, 0, 0);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx4_to_bf16((uint32_t)codes[1], 1.0f), __builtin_bit_cast(bf16x8, w[1]), acc[dt], 0, 0, 0);
      }
    }
  }
  m = m == LOWEST ? LOWEST : MASK ? m : m * p.scale; // natural units

  // the waves' states through LDS
  __syncthreads();
  float* const mo = reinterpret_cast<float*>(lds); // [wave][col][OP]
  float* const sm = mo + W * 16 * OP;              // [wave][col] maximum, then sum
#pragma unroll
  for (int dt = 0; dt < 2 * NJ; dt++)
    if (c < ncol)
      *reinterpret_cast<f32x4*>(mo + (wave * 16 + c) * OP + dt * 16 + g * 4) = acc[dt];
  if (g == 0) {
    sm[wave * 16 + c] = m;
    sm[W * 16 + wave * 16 + c] = sum[0];
  }
  __syncthreads();
  float* const part_o = p.part;
  float* const part_ml = p.part + (int64_t)gridDim.x * p.splits * p.cols * H;
  const int64_t unit = blockIdx.x;
  auto store4 = [&](int cc, int d4, f32x4 v, float Ls) {
    const int cl = o.at * 16 + cc, tk = cl / p.R, rr = cl - tk * p.R;
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; e++) // (nothing seen: zeros; a NaN sum is kept)
      w[e] = f32x2_to_bf16_bits(Ls != 0.f ? v[2 * e] / Ls : 0.f, Ls != 0.f ? v[2 * e + 1] / Ls : 0.f);
    *reinterpret_cast<uint2*>(p.out + ((int64_t)(o.start + tk) * p.Nq + hk * p.R + rr) * H + d4 * 4) = make_uint2(w[0], w[1]);
  };
  for (int i = tid; i < ncol * (H / 4); i += W * 64) {
    const int cc = i / (H / 4), d4 = i % (H / 4);
    float M = sm[cc];
#pragma unroll
    for (int w = 1; w < W; w++)
      M = fmaxf(M, sm[w * 16 + cc]);
    float Ls = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float wt = __builtin_amdgcn_exp2f((sm[w * 16 + cc] - M) * LOG2E);
      Ls = fmaf(wt, sm[W * 16 + w * 16 + cc], Ls);
      const f32x4 ow = *reinterpret_cast<const f32x4*>(mo + (w * 16 + cc) * OP + d4 * 4);
#pragma unroll
      for (int e = 0; e < 4; e++)
        v[e] = fmaf(wt, ow[e], v[e]);
    }
    if (S == 1) {
      store4(cc, d4, v, Ls);
      continue;
    }
    // device-scope stores: written through to the level that all XCDs share
    const int64_t at = (unit * p.splits + blockIdx.y) * p.cols + cc;
    uint64_t* const dst = reinterpret_cast<uint64_t*>(part_o + at * H + d4 * 4);
    __hip_atomic_store(dst, __builtin_bit_cast(uint64_t, make_float2(v[0], v[1])), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(dst + 1, __builtin_bit_cast(uint64_t, make_float2(v[2], v[3])), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (d4 == 0)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(part_ml + at * 2), __builtin_bit_cast(uint64_t, make_float2(M, Ls)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (S == 1)
    return;
  // The split that arrives last merges all of them, in split order (the same sums whichever that is).  Every thread waits until
  // its own stores are acknowledged, then the barrier, the arrival, and the device-scope loads; nobody waits for another workgroup.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    arrived_last = atomicInc(p.counters + unit * MX4_COUNTER_STRIDE, (unsigned)S - 1) == (unsigned)S - 1;
  __syncthreads();
  if (!arrived_last)
    return;
  auto load2 = [](const float* src) {
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(src), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  };
  for (int i = tid; i < ncol * 32; i += W * 64) { // 32 lanes per column, one split each
    const int cc = i >> 5, s = i & 31;
    float2 ml = {LOWEST, 0.f};
    if (s < S)
      ml = load2(part_ml + ((unit * p.splits + s) * p.cols + cc) * 2);
    float M = ml.x;
#pragma unroll
    for (int d = 1; d < 32; d *= 2)
      M = fmaxf(M, __shfl_xor(M, d));
    const float wt = __builtin_amdgcn_exp2f((ml.x - M) * LOG2E);
    float Ls = wt * ml.y;
#pragma unroll
    for (int d = 1; d < 32; d *= 2)
      Ls += __shfl_xor(Ls, d);
    merged[cc][s] = wt;
    if (s == 0)
      merged[cc][32] = Ls;
  }
  __syncthreads();
  for (int i = tid; i < ncol * (H / 4); i += W * 64) {
    const int cc = i / (H / 4), d4 = i % (H / 4);
    const float* src = part_o + (unit * p.splits * p.cols + cc) * H + d4 * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += 8) { // eight splits' loads in flight
      float2 a[8][2];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const float* at = src + (int64_t)min(s0 + u, S - 1) * p.cols * H;
        a[u][0] = load2(at);
        a[u][1] = load2(at + 2);
      }
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (s0 + u < S) {
          const float wt = merged[cc][s0 + u];
          v[0] = fmaf(wt, a[u][0].x, v[0]);
          v[1] = fmaf(wt, a[u][0].y, v[1]);
          v[2] = fmaf(wt, a[u][1].x, v[2]);
          v[3] = fmaf(wt, a[u][1].y, v[3]);
        }
    }
    store4(cc, d4, v, merged[cc][32]);
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int rows_launch(const char* who, Mx4RowsParams& p, bool cache, hipStream_t stream) {
  TPPX_REQUIRE(mx4_has_head(p.H), TPPX_EUNSUPPORTED, "%s: head size %d (64, 96, 128, 192 and 256 are built)", who, p.H);
  TPPX_REQUIRE(p.T >= 0 && p.B > 0 && p.Nkv > 0 && (!p.q || p.Nq > 0) && p.Nq <= (1 << 20) && p.Nkv <= (1 << 20), TPPX_ESHAPE,
               "%s: bad shape T=%d B=%d Nq=%d Nkv=%d", who, p.T, p.B, p.Nq, p.Nkv);
  TPPX_REQUIRE(!p.emb || (p.MP > 0 && p.HR > 0 && p.HR <= p.H && p.HR % 16 == 0), TPPX_ESHAPE,
               "%s: rotary_dim=%d must be a multiple of 16 and <= H=%d", who, p.HR, p.H);
  TPPX_REQUIRE((!p.q || p.q_ld >= (int64_t)p.Nq * p.H) && p.k_ld >= (int64_t)p.Nkv * p.H && (!p.v || p.v_ld >= (int64_t)p.Nkv * p.H) &&
                   (p.q_ld | p.k_ld | p.v_ld) % 8 == 0,
               TPPX_ESHAPE, "%s: row strides must be multiples of 8 elements and hold a row", who);
  if (p.T == 0)
    return TPPX_OK;
  if (!p.emb)
    p.HR = 0;
  const int G = p.H <= 64 ? 4 : p.H <= 128 ? 8 : 16;
  const int64_t rows = (int64_t)(p.q ? p.Nq : 0) + p.Nkv + (p.v ? p.Nkv : 0), blocks = ((int64_t)p.T * G + 255) / 256;
  // Some 1024 workgroups, what the registers let run at once: 2027 tokens of 32 + 2 x 32 heads 21.1 us (5.2 TB/s), 23.6 with 512, 25.3
  // with 4096; 2048 of 64 + 2 x 8 behind the norm 17.3, 19.4, 20.1; without the cache 14.3, 16.3, 15.3.  (A workgroup per token, its
  // heads side by side: 30.6, 27.1 and 18.8, of which the fp64 of the keys was 2.5: rows of the cache were written in pieces by
  // workgroups far apart.)
  const int64_t per_block = std::max<int64_t>(1, std::min<int64_t>({rows, 65535, env_int("TPPX_MX4_ROWS_WGS", 1024) / blocks}));
  const dim3 grid((unsigned)blocks, (unsigned)per_block);
  const bool aligned = p.HR % 64 == 0 && (p.H - p.HR) % 64 == 0;
  auto go = [&](auto g) {
    constexpr int GG = decltype(g)::value;
    if (!cache)
      mx4_rows_kernel<GG, false, true><<<grid, dim3(256), 0, stream>>>(p);
    else if (aligned)
      mx4_rows_kernel<GG, true, true><<<grid, dim3(256), 0, stream>>>(p);
    else
      mx4_rows_kernel<GG, true, false><<<grid, dim3(256), 0, stream>>>(p);
  };
  if (G == 4)
    go(std::integral_constant<int, 4>{});
  else if (G == 8)
    go(std::integral_constant<int, 8>{});
  else
    go(std::integral_constant<int, 16>{});
  return check_hip(hipGetLastError(), who);
}

static int split_launch(const char* who, Mx4AttnParams& p, int H, void* ws, int64_t ws_bytes, void* counters, int64_t counter_bytes,
                        hipStream_t stream) {
  constexpr int W = 4;
  const int64_t blocks = p.cu ? ((int64_t)p.T * p.R + (int64_t)p.B * 15) / 16 : (int64_t)p.B * ((p.R + 15) / 16);
  const int64_t units = blocks * p.Nkv;
  TPPX_REQUIRE(units < ((int64_t)1 << 31), TPPX_ESHAPE, "%s: problem too large", who);
  p.cols = p.cu ? 16 : std::min(16, p.R);
  const int64_t trips = ((int64_t)p.Smax + W * 64 - 1) / (W * 64);
  // 512 workgroups, two per CU (behind a mask and 192 or 256 wide one: 258 registers): 32 x 16000 keys of 8 K/V heads (256 units) 88.5 us with two splits, 93 with three, 105 with four;
  // 8 x 3000 of 16, 256 wide (128) 34 with one, 24.3 with two, 24.7 with four, 27 with twelve; 1 x 2048 of 32 (32) 12.6 with one, 7.8
  // with four, 6.9 with eight; 1 x 16000 of 8 (8) 73 with one, 11.0 with 32; 16 x 2048 of 32 (512) 25.2 with one, 28.9 with two.  Splits
  // beyond a sequence's keys end at once.
  // The merge costs 2 to 4 us, most with 16 columns and many units; a trip over W * 64 keys is about one: split where that saves five
  // trips (24 x 2000 of 8 (192): 15.4 with one split, 16.4 with two; 32 x 500 (256) 7.0 and 8.8; 6 x 12 tokens of 28 heads on 4 behind 1500
  // (148) 12.0, with three 14.6; 64 of 32 heads behind 2000 (128) 16.2, with four 14.4), with single tokens and up to 128 units two
  // (4 x 700 of 16, 256 wide (64) 12.4, with three 8.6; 4 x 1000 of 32 (128) 8.5, with four 8.0).
  // Those were measured in caches as long as their keys.  The lengths are on the device: the rule goes by the capacity, and in a longer
  // cache some short sequences are split where they were better not: 32 x 500 of 8 in 4096 slots 8.5, unsplit 5.8; 16 x 300 of 28 heads on 4 in
  // 4096 7.1 and 5.7; 24 x 2000 of 8 in 4096 15.9 and 14.8.  1 x 2048 of 32 in 16384 takes the 6.7 that it takes in 2112, unsplit 12.6.  A few new
  // tokens gain nothing either: 6 x 7 of 28 heads on 4 behind 1500 12.5 with five splits, unsplit 11.4.
  int64_t S = env_int("TPPX_MX4_SPLITS", 0);
  if (S <= 0) {
    S = std::min<int64_t>(std::max<int64_t>(512 / units, 1), trips);
    if (trips - (trips + S - 1) / S < (p.cu || units > 128 ? 5 : 2))
      S = 1;
  }
  S = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(trips, 32), S));
  if (!ws || units * S * p.cols * (H + 2) * (int64_t)sizeof(float) > ws_bytes || units * MX4_COUNTER_STRIDE * (int64_t)sizeof(unsigned) > counter_bytes)
    S = 1;
  p.splits = (int)S;
  p.part = (float*)ws;
  p.counters = (unsigned int*)counters;
  const dim3 grid((unsigned)units, (unsigned)S);
  // A layer past the 256 MiB of the last-level cache cannot be there from a launch before: its codes go by without being kept (558 MB
  // 102 -> 88.5 us, 6.3 TB/s); smaller ones may be (40 MB 12.3 us, with the hint 13.4; 143 MB 25.2 and 24.8).  This too goes by the
  // capacity: 70 MB of keys in a layer of 285 MB take 13.3 us with the hint, in one of 74 MB 15.1 without it.
  const bool stream_codes = (int64_t)p.B * p.Nkv * p.Smax * H >= ((int64_t)256 << 20);
  mx4_for_head(H, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    auto go = [&](auto m, auto st) {
      mx4_split_kernel<NJ, W, decltype(m)::value, decltype(st)::value><<<grid, dim3(W * 64), 0, stream>>>(p);
    };
    auto with_mask = [&](auto m) {
      if (stream_codes)
        go(m, std::true_type{});
      else
        go(m, std::false_type{});
    };
    if (p.mask)
      with_mask(std::true_type{});
    else
      with_mask(std::false_type{});
  });
  return check_hip(hipGetLastError(), who);
}

static int attn_checks(const char* who, int64_t T, int64_t B, int64_t Nq, int64_t Nkv, int64_t H, int64_t q_ld, const void* mask, int64_t mask_ld) {
  TPPX_REQUIRE(mx4_has_head(H), TPPX_EUNSUPPORTED, "%s: head size %ld (64, 96, 128, 192 and 256 are built)", who, (long)H);
  TPPX_REQUIRE(T >= 0 && T < ((int64_t)1 << 30) && B > 0 && B < ((int64_t)1 << 24) && Nq > 0 && Nkv > 0 && Nq % Nkv == 0 && Nq <= (1 << 16) &&
                   T * (Nq / Nkv) < ((int64_t)1 << 31),
               TPPX_ESHAPE, "%s: bad shape T=%ld B=%ld Nq=%ld Nkv=%ld", who, (long)T, (long)B, (long)Nq, (long)Nkv);
  TPPX_REQUIRE(q_ld >= Nq * H && q_ld % 8 == 0, TPPX_ESHAPE, "%s: row strides must be multiples of 8 elements and hold a row", who);
  TPPX_REQUIRE(!mask || (mask_ld > 0 && mask_ld < ((int64_t)1 << 31)), TPPX_EINVAL, "%s: mask given with mask_ld=%ld", who, (long)mask_ld);
  return TPPX_OK;
}

} // namespace tppx

using namespace tppx;

extern "C" int tppx_qk_norm_rotary(const void* q, const void* k, const void* gamma_q, const void* gamma_k, int gamma_dtype, float eps,
                                   const void* emb_pos, int gptj, const void* pos, void* q_out, void* k_out, int64_t T, int64_t Nq,
                                   int64_t Nkv, int64_t H, int64_t q_ld, int64_t k_ld, int64_t MP, int64_t HR, tppx_stream_t stream) {
  const char* who = "tppx_qk_norm_rotary";
  TPPX_REQUIRE(q && k && q_out && k_out && (pos || !emb_pos), TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(k) && aligned16(q_out) && aligned16(k_out) && aligned16(gamma_q) && aligned16(gamma_k) && aligned16(emb_pos),
               TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  TPPX_REQUIRE(gamma_dtype == TPPX_DT_F32 || gamma_dtype == TPPX_DT_BF16, TPPX_EINVAL, "%s: gamma dtype %d", who, gamma_dtype);
  TPPX_REQUIRE(T < ((int64_t)1 << 31) && MP < ((int64_t)1 << 31) && Nq < (1 << 30) && Nkv < (1 << 30) && H < (1 << 30) && HR < (1 << 30), TPPX_ESHAPE, "%s: problem too large", who);
  Mx4RowsParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k; p.qo = (uint16_t*)q_out; p.ko = (uint16_t*)k_out;
  p.gq = gamma_q; p.gk = gamma_k; p.gamma_f32 = gamma_dtype == TPPX_DT_F32; p.eps = eps;
  p.emb = (const float*)emb_pos; p.gptj = gptj != 0; p.pos = (const int64_t*)pos;
  p.q_ld = q_ld; p.k_ld = k_ld;
  p.T = (int)T; p.B = 1; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.H = (int)H; p.MP = (int)MP; p.HR = (int)HR;
  return rows_launch(who, p, false, (hipStream_t)stream);
}

extern "C" int tppx_append_mx4(const void* q, const void* k, const void* v, const void* gamma_q, const void* gamma_k, int gamma_dtype,
                               float eps, const void* emb_pos, int gptj, const void* pos, void* k_codes, void* k_scales, void* v_codes,
                               void* v_scales, const void* past, const void* cu, void* q_out, void* k_out, void* v_out, int64_t T,
                               int64_t B, int64_t Nq, int64_t Nkv, int64_t H, int64_t Smax, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                               int64_t MP, int64_t HR, tppx_stream_t stream) {
  const char* who = "tppx_append_mx4";
  TPPX_REQUIRE(k && v && k_codes && k_scales && v_codes && v_scales && past && (!q || q_out), TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_out) && aligned16(v_out) && aligned16(gamma_q) &&
                   aligned16(gamma_k) && aligned16(emb_pos) && aligned16(k_codes) && aligned16(v_codes),
               TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  TPPX_REQUIRE(gamma_dtype == TPPX_DT_F32 || gamma_dtype == TPPX_DT_BF16, TPPX_EINVAL, "%s: gamma dtype %d", who, gamma_dtype);
  TPPX_REQUIRE(T < ((int64_t)1 << 31) && B < ((int64_t)1 << 31) && MP < ((int64_t)1 << 31) && Nq < (1 << 30) && Nkv < (1 << 30) && H < (1 << 30) && HR < (1 << 30),
               TPPX_ESHAPE, "%s: problem too large", who);
  TPPX_REQUIRE(Smax > 0 && Smax < ((int64_t)1 << 30), TPPX_ESHAPE, "%s: capacity %ld", who, (long)Smax);
  TPPX_REQUIRE(cu || T == B, TPPX_ESHAPE, "%s: %ld tokens of %ld sequences need their bounds", who, (long)T, (long)B);
  Mx4RowsParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k; p.v = (const uint16_t*)v;
  p.qo = (uint16_t*)q_out; p.ko = (uint16_t*)k_out; p.vo = (uint16_t*)v_out;
  p.kq = (uint8_t*)k_codes; p.ks = (uint8_t*)k_scales; p.vq = (uint8_t*)v_codes; p.vs = (uint8_t*)v_scales;
  p.gq = gamma_q; p.gk = gamma_k; p.gamma_f32 = gamma_dtype == TPPX_DT_F32; p.eps = eps;
  p.emb = (const float*)emb_pos; p.gptj = gptj != 0; p.pos = (const int64_t*)pos;
  p.past = (const int32_t*)past; p.cu = (const int32_t*)cu;
  p.q_ld = q ? q_ld : 0; p.k_ld = k_ld; p.v_ld = v_ld;
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.H = (int)H; p.MP = (int)MP; p.HR = (int)HR; p.Smax = (int)Smax;
  return rows_launch(who, p, true, (hipStream_t)stream);
}

extern "C" int tppx_attn_mx4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                             const void* past, const void* cu, const void* mask, int64_t mask_ld, void* out, int64_t T, int64_t B,
                             int64_t Nq, int64_t Nkv, int64_t H, int64_t Smax, int64_t q_ld, void* ws, int64_t ws_bytes, void* counters,
                             int64_t counter_bytes, tppx_stream_t stream) {
  const char* who = "tppx_attn_mx4";
  TPPX_REQUIRE(q && k_codes && k_scales && v_codes && v_scales && past && out, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(k_codes) && aligned16(v_codes) && aligned16(out) && aligned16(ws), TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  if (int rc = attn_checks(who, T, B, Nq, Nkv, H, q_ld, mask, mask_ld))
    return rc;
  TPPX_REQUIRE(H % 128 != 0 || (((uintptr_t)k_scales | (uintptr_t)v_scales) & (H / 32 - 1)) == 0, TPPX_EINVAL, "%s: scales not aligned to a row of them", who);
  TPPX_REQUIRE(H != 64 || ((uintptr_t)v_scales & 1) == 0, TPPX_EINVAL, "%s: scales not aligned to a row of them", who);
  TPPX_REQUIRE(Smax > 0 && Smax < ((int64_t)1 << 30), TPPX_ESHAPE, "%s: capacity %ld", who, (long)Smax);
  TPPX_REQUIRE(cu || T == B, TPPX_ESHAPE, "%s: %ld tokens of %ld sequences need their bounds", who, (long)T, (long)B);
  TPPX_REQUIRE(ws_bytes >= 0 && (ws_bytes == 0 || ws) && counter_bytes >= 0 && (counter_bytes == 0 || counters), TPPX_EINVAL,
               "%s: size given with a null pointer", who);
  TPPX_REQUIRE(((uintptr_t)counters & 3u) == 0, TPPX_EINVAL, "%s: counters not 4-byte aligned", who);
  if (T == 0)
    return TPPX_OK;
  Mx4AttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const uint16_t*)q; p.q_ld = q_ld;
  p.kq = (const uint8_t*)k_codes; p.ks = (const uint8_t*)k_scales; p.vq = (const uint8_t*)v_codes; p.vs = (const uint8_t*)v_scales;
  p.past = (const int32_t*)past; p.cu = (const int32_t*)cu; p.mask = (const uint16_t*)mask; p.mask_ld = (int)mask_ld; p.out = (uint16_t*)out;
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.R = (int)(Nq / Nkv); p.Smax = (int)Smax;
  p.scale = 1.0f / sqrtf((float)H);
  // The prompt kernel expands a tile of the cache for 128 queries of one head, the split kernel reads it for 16 (token, head) pairs: from
  // enough queries on to fill the chip (T * Nq) the former does less for each, below that its few workgroups walk all keys.  Split
  // kernel and prompt kernel, us: 64 tokens x 64 heads on 8 behind 6000 keys 36 and 120, 256 tokens 94 and 124, 384 133 and 149;
  // 512 x 32 heads behind 2000 46 and 56, 768 66 and 64; 4 x 500 x 12 of 64 19.7 and 22.4; 1200 x 16 of 256 75 and 82.
  // Many sequences of few tokens leave its blocks of queries empty: 32 x 32 tokens x 32 heads 37 and 57, x 48 53 and 68, x 64 67 and 69.
  // (32 columns for a wave of the split kernel, whose expanded operands then serve twice: 512 x 32 heads 45 -> 39, 384 x 64 129 -> 119, below
  // 900 units and from 512 x 64 on slower than what runs there: left out.)
  const int64_t blocks = (T + B * 127) / 128 * Nq;
  if (!cu || (env_int("TPPX_MX4_PROMPT_QUERIES", 0) == 0 && T * Nq * 640 <= 24576 * std::max<int64_t>(640, blocks)))
    return split_launch(who, p, (int)H, ws, ws_bytes, counters, counter_bytes, (hipStream_t)stream);
  return mx4_prompt_launch(who, p, (int)H, true, (hipStream_t)stream);
}

extern "C" int tppx_attn_packed(const void* q, const void* k, const void* v, const void* cu, const void* mask, int64_t mask_ld, void* out,
                                int64_t T, int64_t B, int64_t Nq, int64_t Nkv, int64_t H, int64_t q_ld, int64_t k_ld, int64_t v_ld,
                                tppx_stream_t stream) {
  const char* who = "tppx_attn_packed";
  TPPX_REQUIRE(q && k && v && cu && out, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  if (int rc = attn_checks(who, T, B, Nq, Nkv, H, q_ld, mask, mask_ld))
    return rc;
  TPPX_REQUIRE(k_ld >= Nkv * H && v_ld >= Nkv * H && (k_ld | v_ld) % 8 == 0 && k_ld < (1 << 24) && v_ld < (1 << 24), TPPX_ESHAPE,
               "%s: row strides must be multiples of 8 elements below 2^24 and hold a row", who);
  if (T == 0)
    return TPPX_OK;
  Mx4AttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k; p.v = (const uint16_t*)v; p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld;
  p.cu = (const int32_t*)cu; p.mask = (const uint16_t*)mask; p.mask_ld = (int)mask_ld; p.out = (uint16_t*)out;
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.R = (int)(Nq / Nkv);
  p.scale = 1.0f / sqrtf((float)H);
  return mx4_prompt_launch(who, p, (int)H, false, (hipStream_t)stream);
}
