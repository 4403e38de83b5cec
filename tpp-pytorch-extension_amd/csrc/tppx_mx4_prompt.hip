// Attention of prompts, causal, over packed bf16 rows or over the MXFP4 cache.
#include <algorithm>

#include "tppx_mx4.h"

namespace tppx {

// ---------------------------------------------------------------------------
// In both kernels a workgroup takes the queries of one head in groups, a wave each, which share K and V tiles of 64 (or 32) keys, bf16 in
// LDS in two stages.  Both products run transposed: scores^T[key][query] = K Q^T, out^T[channel][query] += V^T P^T; a lane holds the
// scores of one query, and those, rounded to bf16, are the second operand of the V product as they lie; V's operand is read by the
// transposing LDS read.  Scores in fp32, running maximum and sum per query.
// The sums are relative to a maximum that follows the true one once that is 2^8 above it (the probabilities are then at most 2^8: their
// rounding is relative, and fp32 sums have the room).  Followed at once, nearly every tile rescales: 4 prompts of up to 4100 206 us
// instead of 190 when that was measured.  What it costs is that the largest probability is no longer exactly 1: relative error against
// 64 bits 2.0e-3 there, 1.8e-3 followed at once, 1.65e-3 the rounding of the output alone.  The probabilities' sum is that of the rounded
// ones: where a key outweighs the others its rounding cancels.
// A key that a query does not see (a later token, a mask of -inf) adds nothing whatever it holds: its score is replaced, and in
// tiles where some query misses a key values that are infinite or NaN become zeros in LDS; a workgroup that met such values adds them,
// one by one, to the outputs of the queries that see them once those are written.
// ---------------------------------------------------------------------------
// Values that are not finite, added one by one to what a lane wrote itself: channels d + 4 lane .. + 3 of a row of H, keys from .. limit - 1.
template <int H, int LANES, typename F>
__device__ __forceinline__ void mx4_add_non_finite(uint16_t* orow, int lane, int from, int limit, const uint16_t* mrow, int mask_ld, F&& value) {
#pragma unroll 1
  for (int d = 4 * lane; d < H; d += 4 * LANES) {
    float f[4];
    for (int e = 0; e < 4; e++)
      f[e] = bf16_bits_to_f32(orow[d + e]);
#pragma unroll 1
    for (int key = from; key < limit; key++) {
      if (mrow && key < mask_ld && bf16_bits_to_f32(mrow[key]) == -INFINITY)
        continue;
      for (int e = 0; e < 4; e++) {
        const uint32_t w = value(key, d + e);
        if ((w & 0x7f80u) == 0x7f80u)
          f[e] += bf16_bits_to_f32(w);
      }
    }
    for (int e = 0; e < 4; e++)
      orow[d + e] = (uint16_t)f32_to_bf16_bits(f[e]);
  }
}

// ---------------------------------------------------------------------------
// Over the MXFP4 cache: 128 queries in groups of QW, or with KT = 2 two waves for each group that take half of every tile's keys (and
// are merged at the end: launches of few workgroups).  Codes are expanded once per workgroup on the way to LDS.  32 queries per wave: an
// operand read from LDS feeds 32 columns; heads of 192 and 256 run on 16, for the registers.
// What bounds it: the way of the codes into LDS (without it 35 % less) and, as in the packed kernel, the chain scores, softmax, output
// of a wave (matrix instructions take 0.30 of the time).  512 tokens x 64 heads behind 6000 keys 131 .. 147 us (cards differ), 715 .. 800
// TFLOP/s.
// ---------------------------------------------------------------------------
// Pitch of a row in LDS.  K is read 16 bytes per lane, 16 rows at a time: rows 4 banks apart.  V is read 8 bytes per lane, 4 rows of
// 64 bytes by 32 lanes: rows 16 banks apart (or 48); at K's pitch half of the cycles of LDS were bank conflicts.
// (With 16 queries a wave: 8 rows of 32 bytes by 32 lanes, rows 8 banks apart or an odd multiple of that.)
constexpr int mx4_k_pitch(int NJ) { return 64 * NJ + 16; }
constexpr int mx4_v_pitch(int NJ, int QW) { return QW == 16 ? 64 * NJ + 32 : NJ % 4 == 3 ? 64 * NJ : 64 * NJ + 64; }

template <int NJ, int QW, int KT>
__global__ void __launch_bounds__(128 / QW * KT * 64, 2)
mx4_prompt_kernel(const Mx4AttnParams p) {
  constexpr int QG = 128 / QW; // groups of queries
  constexpr int H = 32 * NJ, KP = mx4_k_pitch(NJ), VP = mx4_v_pitch(NJ, QW), D = 2, STAGE = 64 * (KP + VP); // K rows, then V rows
  // Scores of a lane: NT runs of QW keys of the tile, NV of each, for one query; its output: NA pieces of QW channels.
  constexpr int QB = QW * QG, TH = 64 * QG * KT, NT = 64 / QW / KT, NV = QW / 2 * QW / 32, NA = H / QW, HALF = 64 / QW;
  using Vec = std::conditional_t<QW == 32, f32x16, f32x4>;
  constexpr int PER = NJ, ITEMS = 64 * PER, NC = (ITEMS + TH - 1) / TH; // items of a row, of a tile, of a thread
  extern __shared__ __align__(16) uint8_t lds[]; // 2 stages
  __shared__ int odd_values;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % QG, team = __builtin_amdgcn_readfirstlane(tid >> 6) / QG;
  const int c = lane % QW, h = lane / QW; // query, and group of lanes that share its keys
  // heads go round the XCDs, those of one K/V head to the same one
  const int hr = (int)blockIdx.x % p.Nq, hk = hr % p.Nkv, hq = hk * p.R + hr / p.Nkv;
  // Two workgroups share a CU, and the dispatcher puts workgroup i + 256 beside workgroup i: every other run of whole query blocks
  // within 256 workgroups is walked the other way round, so that a long block meets a short one (2048 tokens x 32 heads, 512
  // workgroups: 69 us without).
  Block o;
  const int run = max(256 / p.Nq, 1);
  const auto paired = [&](int k, int all) {
    const int r = k / run;
    return (r & 1) && (r + 1) * run <= all ? r * run + run - 1 - k % run : k;
  };
  if (!locate(p.cu, p.B, p.T, 1, QB, (int)blockIdx.x / p.Nq, o, paired))
    return;
  const int qblk = (o.n + QB - 1) / QB - 1 - o.at; // the last queries see the most keys: first
  const int past = mx4_past(p.past[o.b], p.Smax);
  const int total = min(past + o.n, p.Smax); // keys of the sequence
  const int q0 = qblk * QB + wave * QW;
  const int qi = min(q0 + c, o.n - 1);
  const int limit = min(past + qi + 1, total); // keys this lane's query sees
  const int64_t head = ((int64_t)o.b * p.Nkv + hk) * p.Smax;
  const uint8_t* const kq = p.kq + head * (16 * NJ);
  const uint8_t* const vq = p.vq + head * (16 * NJ);
  const uint8_t* const ks = p.ks + head * NJ;
  const uint8_t* const vs = p.vs + head * NJ;
  const uint16_t* const mrow = p.mask ? p.mask + (int64_t)o.b * p.mask_ld : nullptr;

  constexpr int NK = H / (8 * HALF); // steps of the score's sum
  bf16x8 q[NK];
  {
    const uint16_t* qrow = p.q + (int64_t)(o.start + qi) * p.q_ld + (int64_t)hq * H + h * 8;
#pragma unroll
    for (int j = 0; j < NK; j++)
      q[j] = *reinterpret_cast<const bf16x8*>(qrow + j * (8 * HALF));
  }
  // keys that some query of this workgroup sees
  const int keys = min(past + min(qblk * QB + QB, o.n), total), tiles = (keys + 63) / 64;
  const int first_limit = min(past + qblk * QB + 1, total); // keys that all of them see

  // Item i of thread tid: a block of a row of K (V false) or of V; rows past the keys: zeros.  They pass through registers, asked for two
  // tiles before they are expanded on the way to LDS (2048 tokens behind 2048 124 us, one tile before 132).
  i32x4 k_item[D][NC], v_item[D][NC];
  uint32_t k_byte[D][NC], v_byte[D][NC];
  // (buffers of a tile's rows: what lies past them reads as zero, with no branch and no access)
  auto request = [&](auto V_, auto S_, int kb) {
    constexpr bool V = decltype(V_)::value;
    constexpr int slot = decltype(S_)::value % D;
    auto& item = V ? v_item[slot] : k_item[slot];
    auto& byte = V ? v_byte[slot] : k_byte[slot];
    const int rows = min(max(keys - kb * 64, 0), 64);
    auto rsrc = [](const void* at, uint32_t bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, (int)bytes, 0x00020000);
    };
    const auto codes = rsrc((V ? vq : kq) + (int64_t)kb * (64 * 16 * NJ), rows * (16 * NJ));
    const auto scales = rsrc((V ? vs : ks) + (int64_t)kb * (64 * NJ), rows * NJ);
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int at = i * TH + tid;
      item[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, at * 16, 0, 0));
      byte[i] = __builtin_amdgcn_raw_buffer_load_b8(scales, at, 0, 0);
    }
  };
  auto chunk_of = [](const i32x4& w, int j) { // (no indexed registers)
    const int lo = j & 1 ? w[1] : w[0], hi = j & 1 ? w[3] : w[2];
    return j & 2 ? hi : lo;
  };
  auto turn_of = [](int row) { return QW == 16 ? (row >> 1) & 3 : row & 3; };
  auto deliver = [&](auto V_, auto S_, int kb) {
    constexpr bool V = decltype(V_)::value;
    constexpr int stage = decltype(S_)::value, slot = stage % D;
    auto& item = V ? v_item[slot] : k_item[slot];
    auto& byte = V ? v_byte[slot] : k_byte[slot];
    uint8_t* const st = lds + stage * STAGE + (V ? 64 * KP : 0);
    constexpr int PITCH = V ? VP : KP;
    const bool partial = V && (mrow || kb * 64 + 64 > first_limit); // (uniform)
    bool odd = false;
#pragma unroll
    for (int i = 0; i < NC; i++) {
      const int at = i * TH + tid, row = at / PER, ch = at % PER;
      uint8_t* const dst = st + row * PITCH + ch * 64;
      if (ITEMS % TH == 0 || at < ITEMS) {
        const bool nan = byte[i] == 255u, drop = nan && partial;
        odd |= drop;
        const float s = e8m0_to_f32(drop ? 0u : byte[i]);
#pragma unroll
        for (int j = 0; j < 4; j++) // (V's rows are 16 banks apart, as a block's chunks are: another order of them in each row)
          *reinterpret_cast<bf16x8*>(dst + (V ? (j ^ turn_of(row)) * 16 : j * 16)) =
              mx4_to_bf16(nan ? 0u : (uint32_t)(V ? chunk_of(item[i], j ^ turn_of(row)) : item[i][j]), s); // (zero times infinity)
      }
    }
    if (odd)
      odd_values = 1;
  };
  constexpr std::false_type K_{};
  constexpr std::true_type V_{};

  float m = LOWEST, l = 0.f;
  Vec acc[NA];
#pragma unroll
  for (int dt = 0; dt < NA; dt++)
#pragma unroll
    for (int i = 0; i < NV; i++)
      acc[dt][i] = 0.f;
  const float scale2 = p.scale * LOG2E;
  const int wave_limit = min(past + min(q0 + QW, o.n), total); // keys that some query of this wave sees
  const bool idle = q0 >= o.n;

  if (tid == 0)
    odd_values = 0;
  constexpr std::integral_constant<int, 0> EVEN{};
  constexpr std::integral_constant<int, 1> ODD{};
  request(K_, EVEN, 0);
  request(V_, EVEN, 0);
  request(K_, ODD, 1);
  request(V_, ODD, 1);
  __syncthreads();
  deliver(K_, EVEN, 0);
  request(K_, EVEN, D);
  deliver(V_, EVEN, 0);
  request(V_, EVEN, D);
  auto turn = [&](auto S_, int kb) { // tile kb, in stage kb & 1
    constexpr int stage = decltype(S_)::value;
    constexpr std::integral_constant<int, stage ^ 1> NEXT{};
    __syncthreads(); // this tile has been written, the other stage has been read
    const bool more = kb + 1 < tiles, busy = !idle && kb * 64 < wave_limit; // (uniform in a wave)
    const uint8_t* const st = lds + stage * STAGE;
    bf16x8 pb[NT * NV / 8];
    Vec sc[NT];
    if (busy) {
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < NV; i++)
          sc[t][i] = 0.f;
#pragma unroll
        for (int j = 0; j < NK; j++) {
          const bf16x8 w = *reinterpret_cast<const bf16x8*>(st + (team * 32 + t * QW + c) * KP + (j * HALF + h) * 16);
          if constexpr (QW == 32)
            sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, q[j], sc[t], 0, 0, 0);
          else
            sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, q[j], sc[t], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (KT == 1 && more) { // under the matrix instructions (with half of them it comes better behind the softmax)
      deliver(K_, NEXT, kb + 1);
      request(K_, NEXT, kb + 1 + D);
    }
    if (busy) {
      // key of score i of run t
      auto key_of = [&](int t, int i) { return kb * 64 + team * 32 + t * QW + (QW == 32 ? (i & 3) + 8 * (i >> 2) : i) + 4 * h; };
      if (mrow) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < NV; i++) {
            const int key = key_of(t, i);
            const float mv = key < p.mask_ld ? bf16_bits_to_f32(mrow[min(key, p.mask_ld - 1)]) : 0.f;
            sc[t][i] = mv == -INFINITY ? -INFINITY : fmaf(sc[t][i], p.scale, mv);
          }
      }
      const bool partial = kb * 64 + 64 > min(past + q0 + 1, total); // (wave-uniform)
      if (partial) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < NV; i++)
            sc[t][i] = key_of(t, i) < limit ? sc[t][i] : -INFINITY;
      }
      float mx = m;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < NV; i++)
          mx = fmaxf(mx, sc[t][i]);
      const float unit = mrow ? LOG2E : scale2;
      float alpha = 1.f;
      if (__builtin_amdgcn_ballot_w64((mx - m) * unit > 8.f) != 0) {
        if constexpr (QW == 16) {
          mx = max_of_groups(mx);
        } else {
          auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        alpha = __builtin_amdgcn_exp2f((m - mx) * unit);
#pragma unroll
        for (int dt = 0; dt < NA; dt++)
          acc[dt] *= alpha;
        m = mx;
      }
      l *= alpha;
      float off = -m * unit;
      if (mrow) { // (the difference first: a mask's lowest value times log2 e is no number)
        off = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++)
          sc[t] -= m;
      }
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < NV; i += 2) {
          const bf16x2 pr = {(__bf16)__builtin_amdgcn_exp2f(fmaf(sc[t][i], unit, off)), (__bf16)__builtin_amdgcn_exp2f(fmaf(sc[t][i + 1], unit, off))};
          l = __builtin_amdgcn_fdot2_f32_bf16(pr, bf16x2{(__bf16)1.f, (__bf16)1.f}, l, false);
          pb[(t * NV + i) >> 3][(t * NV + i) & 7] = pr[0];
          pb[(t * NV + i) >> 3][((t * NV + i) & 7) + 1] = pr[1];
        }
    }
    if (KT != 1 && more) {
      deliver(K_, NEXT, kb + 1);
      request(K_, NEXT, kb + 1 + D);
    }
    if (busy) {
      // V operand of the keys of a P operand and QW channels: two transposing reads of 4 keys each for this lane's group (32 queries a
      // wave: 16 keys, 8 apart; 16: 32 keys, 16 apart)
      constexpr int KEYS = QW == 32 ? 16 : 32;
      const uint8_t* const vt = st + 64 * KP + (team * 32 + 4 * h + ((lane & 15) >> 2)) * VP + (QW == 32 ? ((lane >> 4) & 1) * 32 : 0) + (lane & 3) * 8;
      auto operand = [&](int dt, int u, int e) {
        return __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(vt + (u * KEYS + e * (KEYS / 2)) * VP + dt * (2 * QW))));
      };
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < NT * NV / 8; u++)
#pragma unroll
        for (int dt = 0; dt < NA; dt++) {
          const i32x2 a = operand(dt, u, 0), b = operand(dt, u, 1);
          const bf16x8 w = __builtin_bit_cast(bf16x8, i32x4{a[0], a[1], b[0], b[1]});
          if constexpr (QW == 32)
            acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, pb[u], acc[dt], 0, 0, 0);
          else
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, pb[u], acc[dt], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (more) {
      deliver(V_, NEXT, kb + 1);
      request(V_, NEXT, kb + 1 + D);
    }
  };
  for (int kb = 0; kb < tiles; kb += 2) {
    turn(EVEN, kb);
    if (kb + 1 < tiles)
      turn(ODD, kb + 1);
  }
  if constexpr (QW == 16)
    l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if constexpr (KT > 1) { // the second team's state through LDS
    float* const at = reinterpret_cast<float*>(lds) + (wave * 64 + lane) * 4;
    constexpr int STEP = QG * 64 * 4;
    const float unit = mrow ? LOG2E : scale2;
    __syncthreads(); // the stages have been read
    if (team) {
#pragma unroll
      for (int k = 0; k < 4 * NJ; k++)
        *reinterpret_cast<f32x4*>(at + k * STEP) = f32x4{acc[k >> 2][(k & 3) * 4], acc[k >> 2][(k & 3) * 4 + 1], acc[k >> 2][(k & 3) * 4 + 2], acc[k >> 2][(k & 3) * 4 + 3]};
      at[4 * NJ * STEP] = m;
      at[4 * NJ * STEP + 1] = l;
    }
    __syncthreads();
    if (team)
      return;
    const float m1 = at[4 * NJ * STEP], mm = fmaxf(m, m1);
    const float a = __builtin_amdgcn_exp2f((m - mm) * unit), b = __builtin_amdgcn_exp2f((m1 - mm) * unit);
    l = l * a + at[4 * NJ * STEP + 1] * b;
#pragma unroll
    for (int k = 0; k < 4 * NJ; k++) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(at + k * STEP);
#pragma unroll
      for (int e = 0; e < 4; e++)
        acc[k >> 2][(k & 3) * 4 + e] = acc[k >> 2][(k & 3) * 4 + e] * a + v[e] * b;
    }
  }
  if (q0 + c < o.n) {
    uint16_t* orow = p.out + ((int64_t)(o.start + q0 + c) * p.Nq + hq) * H;
    const float inv = l != 0.f ? 1.0f / l : 0.f; // (nothing seen: zeros)
#pragma unroll
    for (int dt = 0; dt < NA; dt++)
#pragma unroll
      for (int i = 0; i < NV; i += 4) {
        const uint2 w = make_uint2(f32x2_to_bf16_bits(acc[dt][i] * inv, acc[dt][i + 1] * inv), f32x2_to_bf16_bits(acc[dt][i + 2] * inv, acc[dt][i + 3] * inv));
        *reinterpret_cast<uint2*>(orow + dt * QW + 8 * (i >> 2) + 4 * h) = w;
      }
    if (__builtin_expect(odd_values != 0, 0))
      mx4_add_non_finite<H, HALF>(orow, h, mrow ? 0 : max(first_limit, 0) / 64 * 64, limit, mrow, p.mask_ld,
                                  [&](int key, int ch) { return vs[(int64_t)key * NJ + (ch >> 5)] == 255 ? 0x7fc0u : 0u; });
  }
}

// ---------------------------------------------------------------------------
// Packed bf16 prompts: W waves of 16 queries, tiles of KEYS keys brought by loads straight into LDS, one ahead.  The chunks of 16 bytes
// of a row lie permuted (those loads write 1024 bytes in a row), so that neither the rows of a K operand nor the pieces that the
// transposing read of V takes meet in a bank.
// A value that is infinite where a query sees it but its probability is below fp32's range gives NaN by the matrix instruction in
// whole tiles (zero times infinity) and its infinity in those that end inside the sequence, where it is added by itself.
// What bounds it: the chain scores, softmax, output of a wave (matrix instructions take 0.39 of the time); so four waves per SIMD in 128
// registers count for more than operands that feed 32 queries.  Measured against 32 queries a wave, two per SIMD, the tiles through
// registers: 4 prompts of up to 4100 tokens x 32 heads 187 -> 171 us (on other cards 161 .. 183, 800 .. 910 TFLOP/s, where a large library
// product reaches 1138 .. 1417), 2048 x
// 32 heads 64 -> 52, 2048 x 64 on 8 95 -> 85, 2048 x 16 of 256 93 -> 77, 333 x 32 12.7 -> 10.6, 4 x 1000 x 12 of 64 28 -> 24.
// Tried in that other form and slower: this tile's output and the next one's scores as one sequence of independent matrix
// instructions (219 where it took 190), 256 queries in eight waves (195).
// ---------------------------------------------------------------------------
template <int NJ, int W, int KEYS>
__global__ void __launch_bounds__(W * 64, NJ == 4 && (W == 8 || KEYS == 32) ? 4 : 2)
mx4_packed_kernel(const Mx4AttnParams p) {
  constexpr int H = 32 * NJ, ROW = 64 * NJ, PER = 4 * NJ, SIDE = KEYS * ROW, QB = 16 * W, TH = 64 * W, NA = H / 16;
  // Addresses of operands that differ in the turn of their chunks (the others lie at fixed distances), pieces of V per read.
  constexpr int XK = NJ % 4 == 0 ? 4 : NJ % 2 == 0 ? 2 : 1, XV = NJ % 4 == 0 ? 8 : NJ % 2 == 0 ? 4 : 2, NR = NJ == 3 ? 6 : XV;
  extern __shared__ __align__(16) uint8_t lds[]; // V of two stages, then K
  __shared__ int odd_values;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int hr = (int)blockIdx.x % p.Nq, hk = hr % p.Nkv, hq = hk * p.R + hr / p.Nkv;
  Block o;
  const int run = max(256 / p.Nq, 1);
  const auto paired = [&](int k, int all) {
    const int r = k / run;
    return (r & 1) && (r + 1) * run <= all ? r * run + run - 1 - k % run : k;
  };
  if (!locate(p.cu, p.B, p.T, 1, QB, (int)blockIdx.x / p.Nq, o, paired))
    return;
  const int qblk = (o.n + QB - 1) / QB - 1 - o.at; // the last queries see the most keys: first
  const int q0 = qblk * QB + wave * 16;
  const int qi = min(q0 + c, o.n - 1); // this lane's query: sees the keys 0 .. qi
  const uint16_t* const kr = p.k + (int64_t)o.start * p.k_ld + hk * H;
  const uint16_t* const vr = p.v + (int64_t)o.start * p.v_ld + hk * H;
  const uint16_t* const mrow = p.mask ? p.mask + (int64_t)o.b * p.mask_ld : nullptr;
  bf16x8 q[NJ];
  {
    const uint16_t* qrow = p.q + (int64_t)(o.start + qi) * p.q_ld + (int64_t)hq * H + g * 8;
#pragma unroll
    for (int j = 0; j < NJ; j++)
      q[j] = *reinterpret_cast<const bf16x8*>(qrow + j * 32);
  }
  const int keys = min(qblk * QB + QB, o.n), tiles = (keys + KEYS - 1) / KEYS; // keys that some query of this workgroup sees
  const int first_limit = qblk * QB + 1;                              // keys that all of them see

  // Pieces of 1024 bytes: KEYS / 16 waves bring K, NJ pieces each, and as many V, others or the same.
  constexpr int SW = KEYS / 16, SIDES = W == SW ? 2 : 1;
  uint32_t from[SIDES][NJ]; // offset of this lane's chunk in the tile's rows
  auto side_of = [&](int s) { return SIDES == 1 ? wave / SW : s; }; // 1: V
  auto offset = [&](int s, int i, int rows) {
    const int item = (wave % SW * NJ + i) * 64 + lane, row = item / PER, ch = item % PER;
    const int turn = side_of(s) ? packed_v_turn(NJ, row) : packed_k_turn(NJ, row);
    return ((uint32_t)min(row, rows - 1) * (uint32_t)(side_of(s) ? p.v_ld : p.k_ld) + (uint32_t)(ch ^ turn) * 8u) * 2u;
  };
#pragma unroll
  for (int s = 0; s < SIDES; s++)
#pragma unroll
    for (int i = 0; i < NJ; i++)
      from[s][i] = offset(s, i, KEYS);
  auto request = [&](int kb, int stage) {
    const int rows = min(keys - kb * KEYS, KEYS);
#pragma unroll
    for (int s = 0; s < SIDES; s++) {
      const int64_t ld = side_of(s) ? p.v_ld : p.k_ld;
      const auto src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>((side_of(s) ? vr : kr) + (int64_t)kb * KEYS * ld), 0,
                                                         (int)(((uint32_t)(rows - 1) * (uint32_t)ld + H) * 2u), 0x00020000);
      uint8_t* const dst = lds + (side_of(s) ? 0 : 2 * SIDE) + stage * SIDE + wave % SW * (NJ * 1024);
#pragma unroll
      for (int i = 0; i < NJ; i++) { // (rows past the keys repeat the last one)
        const uint32_t at = rows < KEYS ? offset(s, i, rows) : from[s][i];
        load_to_lds(src, dst + i * 1024, at);
      }
    }
  };
  uint32_t kaddr[XK], vaddr[XV];
#pragma unroll
  for (int j = 0; j < XK; j++)
    kaddr[j] = (uint32_t)(2 * SIDE + c * ROW + ((j * 4 + g) ^ packed_k_turn(NJ, c)) * 16);
  {
    const int r = g * 4 + (c >> 2);
#pragma unroll
    for (int d = 0; d < XV; d++)
      vaddr[d] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds + (uint32_t)(r * ROW + ((d * 2 + ((c >> 1) & 1)) ^ packed_v_turn(NJ, r)) * 16 + (c & 1) * 8);
  }

  float m, l;
  f32x4 acc[NA];
  // Values that are not finite leave V (in LDS) where some query may not see them.  Four waves on tiles of 64 keys look for them only once
  // a sum came out infinite or NaN, in a second run over the tiles (333 tokens x 32 heads 11.0 -> 10.4 us, 2 masked prompts of 700 41 -> 36);
  // the other forms look in the first (the second run's registers are more than 128: 52 -> 56 us for 2048).
  bool careful = NJ >= 4 && (W == 8 || KEYS == 32);
  const float unit = mrow ? LOG2E : p.scale * LOG2E;
  if (tid == 0)
    odd_values = 0;
  auto tile = [&](auto S_, int kb) {
    constexpr int stage = decltype(S_)::value;
    // this tile has landed and the other stage has been read, for this wave and then for every wave
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
    if (careful && (mrow || kb * KEYS + KEYS > first_limit)) { // (uniform) some query may not see some key
      bool odd = false;
#pragma unroll
      for (int i = 0; i < (KEYS * PER + TH - 1) / TH; i++) {
        const int at = i * TH + tid;
        if (KEYS * PER % TH == 0 || at < KEYS * PER) {
          i32x4* const it = reinterpret_cast<i32x4*>(lds + stage * SIDE) + at;
          const i32x4 w = *it;
          bool some = false;
#pragma unroll
          for (int j = 0; j < 4; j++)
            some |= mx4_non_finite((uint32_t)w[j]);
          if (some)
            *it = i32x4{(int)mx4_finite((uint32_t)w[0]), (int)mx4_finite((uint32_t)w[1]), (int)mx4_finite((uint32_t)w[2]), (int)mx4_finite((uint32_t)w[3])};
          odd |= some;
        }
      }
      if (odd)
        odd_values = 1;
      __syncthreads();
    }
    if (kb + 1 < tiles)
      request(kb + 1, stage ^ 1); // in flight during the arithmetic below
    if (kb * KEYS > min(q0 + 15, o.n - 1) || q0 >= o.n)
      return; // past what this wave's queries see
    const uint8_t* const st = lds + stage * SIDE;
    constexpr int NT = KEYS / 16; // runs of 16 keys
    f32x4 sc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; j++)
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(st + kaddr[j % XK] + t * (16 * ROW) + j / XK * (XK * 64)), q[j], sc[t], 0, 0, 0);
    }
    if (mrow) {
#pragma unroll
      for (int i = 0; i < 4 * NT; i++) {
        const int key = kb * KEYS + (i >> 2) * 16 + g * 4 + (i & 3);
        const float mv = key < p.mask_ld ? bf16_bits_to_f32(mrow[min(key, p.mask_ld - 1)]) : 0.f;
        sc[i >> 2][i & 3] = mv == -INFINITY ? -INFINITY : fmaf(sc[i >> 2][i & 3], p.scale, mv);
      }
    }
    if (kb * KEYS + KEYS - 1 > q0) { // (wave-uniform)
#pragma unroll
      for (int i = 0; i < 4 * NT; i++)
        sc[i >> 2][i & 3] = kb * KEYS + (i >> 2) * 16 + g * 4 + (i & 3) <= qi ? sc[i >> 2][i & 3] : -INFINITY;
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < 4 * NT; i++)
      mx = fmaxf(mx, sc[i >> 2][i & 3]);
    if (__builtin_amdgcn_ballot_w64((mx - m) * unit > 8.f) != 0) {
      mx = max_of_groups(mx);
      const float alpha = __builtin_amdgcn_exp2f((m - mx) * unit);
#pragma unroll
      for (int dt = 0; dt < NA; dt++)
        acc[dt] *= alpha;
      l *= alpha;
      m = mx;
    }
    float off = -m * unit;
    if (mrow) { // (the difference first: a mask's lowest value times log2 e is no number)
      off = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++)
        sc[t] -= m;
    }
    bf16x8 pb[KEYS / 32];
#pragma unroll
    for (int i = 0; i < 4 * NT; i += 2) {
      const bf16x2 pr = {(__bf16)__builtin_amdgcn_exp2f(fmaf(sc[i >> 2][i & 3], unit, off)), (__bf16)__builtin_amdgcn_exp2f(fmaf(sc[i >> 2][(i & 3) + 1], unit, off))};
      l = __builtin_amdgcn_fdot2_f32_bf16(pr, bf16x2{(__bf16)1.f, (__bf16)1.f}, l, false);
      pb[i >> 3][i & 7] = pr[0];
      pb[i >> 3][(i & 7) + 1] = pr[1];
    }
    static_for<0, KEYS / 32 * (NA / NR)>([&](auto I) { // 32 keys, NR pieces of channels
      constexpr int u = decltype(I)::value / (NA / NR), d0 = decltype(I)::value % (NA / NR) * NR;
      i32x2 vv[NR][2];
      packed_v_operands<stage * SIDE + u * 32 * ROW + d0 * 32, 16 * ROW>(vv, vaddr);
#pragma unroll
      for (int d = 0; d < NR; d++) {
        const i32x4 w = {vv[d][0][0], vv[d][0][1], vv[d][1][0], vv[d][1][1]};
        acc[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), pb[u], acc[d0 + d], 0, 0, 0);
      }
    });
  };
  for (;;) {
    m = LOWEST;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < NA; dt++)
      acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    request(0, 0);
    for (int kb = 0; kb < tiles; kb += 2) {
      tile(std::integral_constant<int, 0>{}, kb);
      if (kb + 1 < tiles)
        tile(std::integral_constant<int, 1>{}, kb + 1);
    }
    if (careful)
      break;
    f32x4 none = {0.f, 0.f, 0.f, 0.f}; // NaN where a sum is infinite or NaN
#pragma unroll
    for (int dt = 0; dt < NA; dt++)
      none += acc[dt] * 0.f;
    if (!__syncthreads_or(!(none[0] + none[1] + none[2] + none[3] == 0.f)))
      break;
    careful = true; // once more: an unseen value may be among them
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (q0 + c < o.n) {
    uint16_t* orow = p.out + ((int64_t)(o.start + q0 + c) * p.Nq + hq) * H;
    const float inv = l != 0.f ? 1.0f / l : 0.f; // (nothing seen: zeros)
#pragma unroll
    for (int dt = 0; dt < NA; dt++)
      *reinterpret_cast<uint2*>(orow + dt * 16 + g * 4) =
          make_uint2(f32x2_to_bf16_bits(acc[dt][0] * inv, acc[dt][1] * inv), f32x2_to_bf16_bits(acc[dt][2] * inv, acc[dt][3] * inv));
    if (__builtin_expect(odd_values != 0, 0))
      mx4_add_non_finite<H, 4>(orow, g, mrow ? 0 : first_limit / KEYS * KEYS, qi + 1, mrow, p.mask_ld, [&](int key, int ch) { return (uint32_t)vr[(int64_t)key * p.v_ld + ch]; });
  }
}

int mx4_prompt_launch(const char* who, const Mx4AttnParams& p, int H, bool cache, hipStream_t stream) {
  // every sequence's last workgroup may be short: at most this many, those past the last one end at once
  auto blocks = [&](int rows) { return ((int64_t)p.T + (int64_t)p.B * (rows - 1)) / rows * p.Nq; };
  const int form = env_int("TPPX_MX4_PROMPT_QUERIES", 0);
  const bool many = form ? form >= 128 : blocks(128) >= (H > 128 ? 200 : 400);
  hipError_t e = hipSuccess;
  int rc = TPPX_OK;
  auto go = [&](auto kern, int rows, int threads, size_t lds) {
    const int64_t wgs = blocks(rows);
    if (wgs >= ((int64_t)1 << 31)) {
      rc = set_error(TPPX_ESHAPE, "%s: problem too large", who);
      return;
    }
    e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds);
    if (e == hipSuccess)
      kern<<<dim3((unsigned)wgs), dim3(threads), lds, stream>>>(p);
  };
  mx4_for_head(H, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    if (!cache) {
      // Heads of 64 and 96: 64 queries in four waves (24 x 50..500 tokens x 12 heads of 64 12.0 us, of 128 in eight 14.5; 4000 x 12 48 and 54; 4 x
      // 4000 x 10 of 96 171 and 175).  Wider ones in launches of some 400 (200 beyond 128 wide) workgroups of 128 queries and more: those
      // (2048 tokens x 32 heads, 512: 51, of 64 57; 2048 x 16 heads of 256, 256: 77 and 91; 1000 x 32 heads, 256: 25.3 and 23.1; 333 x 32 11.5
      // and 10.6), and where the prompts are short on average 64 queries on tiles of 32 keys, of whose workgroups four (128 wide; 192 three, 256 two) run on a CU
      // (16 x 17..200 x 28 heads 13.3 -> 11.8, 8 x 50..500 x 64 on 8 31.3 -> 28.7, 16 x 300 x 32 41 -> 38, 16 x 300 x 16 of 256 33.0 -> 30.7; 4 x 1000 x 64 on
      // 8 95 and 101, 6 x 60..1500 x 32 43.5 and 45.9).
      constexpr size_t lds = 4 * 64 * 64 * (size_t)NJ;
      if constexpr (NJ >= 4) {
        if (many && !form && p.T < (int64_t)512 * p.B) {
          go(mx4_packed_kernel<NJ, 4, 32>, 64, 256, lds / 2);
          return;
        }
        if (many) {
          go(mx4_packed_kernel<NJ, 8, 64>, 128, 512, lds);
          return;
        }
      }
      go(mx4_packed_kernel<NJ, 4, 64>, 64, 256, lds);
      return;
    }
    auto over = [&](auto qw, auto kt) {
      constexpr int QW = decltype(qw)::value, KT = decltype(kt)::value, QG = 128 / QW;
      const size_t stages = 2 * 64 * (size_t)(mx4_k_pitch(NJ) + mx4_v_pitch(NJ, QW)), teams = KT > 1 ? QG * 64 * 16 * (size_t)(4 * NJ + 1) : 0;
      go(mx4_prompt_kernel<NJ, QW, KT>, 128, QG * KT * 64, std::max(stages, teams)); // (the state of a second team)
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    // 192 and 256 wide: one workgroup's tiles fill the LDS of a CU, and 32 queries a wave its registers at one wave per SIMD; with 16
    // queries two fit.  Others: 128 queries in four waves, two workgroups on a CU, from 400 of them on, below that two teams that halve the
    // way through a tile (512 tokens x 64 heads behind 6000 keys, 256: 134 us, 167 with one team).  Eight waves of 16 queries that expand
    // into the layout of the packed kernel, with one team or two, were no faster (158 and 134 there; 1024 tokens 246 and 277, here 235).
    if constexpr (NJ > 4)
      over(std::integral_constant<int, 16>{}, one);
    else if (many)
      over(std::integral_constant<int, 32>{}, one);
    else
      over(std::integral_constant<int, 32>{}, two);
  });
  if (rc)
    return rc;
  return check_hip(e != hipSuccess ? e : hipGetLastError(), who);
}
} // namespace tppx
