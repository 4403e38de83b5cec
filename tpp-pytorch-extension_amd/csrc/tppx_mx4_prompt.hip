// Attention of prompts, causal, over packed bf16 rows or over the MXFP4 cache.
#include <algorithm>

#include "tppx_mx4.h"

namespace tppx {

// ---------------------------------------------------------------------------
// Prompts: QG groups of QW queries of one head, each a wave, or with KT = 2 two that take half of every tile's keys (and are
// merged at the end: launches of few workgroups), share K and V tiles of 64 keys, bf16 in LDS in two stages, from packed rows or
// from the cache (its codes expanded once per workgroup on the way to LDS).  Both products run transposed on the QW x QW MFMA:
// scores^T[key][query] = K Q^T, out^T[channel][query] += V^T P^T; a lane holds the scores of one query, and those, rounded to bf16,
// are the second operand of the V product as they lie; V's operand is read by the transposing LDS read.
// 32 queries per wave: an operand read from LDS feeds 32 columns, with 16 the LDS (128 bytes per cycle) takes twice the MFMAs' time;
// heads of 192 and 256 run on 16, for the registers.  Scores in fp32, running maximum and sum per query.
// What bounds it: matrix instructions take a third of the time (4 prompts of up to 4100 tokens x 32 heads 183 us, 800 TFLOP/s, where a
// large library product reaches 1138), the vector instructions of the softmax as much, LDS a quarter; two waves per SIMD overlap them
// in part.  With neither exponentials nor sums it ran 10 % faster, without loads 14 %, without the way into LDS 6 % (over the cache,
// where that expands the codes, 35 %).  Tried and slower: this tile's output and the next one's scores as one sequence of independent
// matrix instructions (219), 256 queries in eight waves (195).
// A key that a query does not see (a later token, a mask of -inf) adds nothing whatever it holds: its score is replaced, and in
// tiles where some query misses a key values that are infinite or NaN become zeros on the way to LDS; a workgroup that met
// such values adds them, one by one, to the outputs of the queries that see them once those are written.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool mx4_non_finite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}
// the pair with what is not finite set to zero
__device__ __forceinline__ uint32_t mx4_finite(uint32_t pair) {
  return ((pair & 0x7f80u) == 0x7f80u ? 0u : pair & 0xffffu) | ((pair & 0x7f800000u) == 0x7f800000u ? 0u : pair & 0xffff0000u);
}

// Pitch of a row in LDS.  K is read 16 bytes per lane, 16 rows at a time: rows 4 banks apart.  V is read 8 bytes per lane, 4 rows of
// 64 bytes by 32 lanes: rows 16 banks apart (or 48); at K's pitch half of the cycles of LDS were bank conflicts.
// (With 16 queries a wave: 8 rows of 32 bytes by 32 lanes, rows 8 banks apart or an odd multiple of that.)
constexpr int mx4_k_pitch(int NJ) { return 64 * NJ + 16; }
constexpr int mx4_v_pitch(int NJ, int QW) { return QW == 16 ? 64 * NJ + 32 : NJ % 4 == 3 ? 64 * NJ : 64 * NJ + 64; }

template <int NJ, int QW, int QG, int KT, bool CACHE>
__global__ void __launch_bounds__(QG * KT * 64, QW == 16 ? (NJ <= 4 && QG == 8 ? 4 : 2) : NJ > 4 ? 1 : 2)
mx4_prompt_kernel(const Mx4AttnParams p) {
  constexpr int H = 32 * NJ, KP = mx4_k_pitch(NJ), VP = mx4_v_pitch(NJ, QW), D = CACHE ? 2 : 1, STAGE = 64 * (KP + VP); // K rows, then V rows
  // Scores of a lane: NT runs of QW keys of the tile, NV of each, for one query; its output: NA pieces of QW channels.
  constexpr int QB = QW * QG, TH = 64 * QG * KT, NT = 64 / QW / KT, NV = QW / 2 * QW / 32, NA = H / QW, HALF = 64 / QW;
  using Vec = std::conditional_t<QW == 32, f32x16, f32x4>;
  constexpr int PER = CACHE ? NJ : 4 * NJ, ITEMS = 64 * PER, NC = (ITEMS + TH - 1) / TH; // items of a row, of a tile, of a thread
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
  const int past = CACHE ? max(p.past[o.b], 0) : 0;
  const int total = CACHE ? min(past + o.n, p.Smax) : o.n; // keys of the sequence
  const int q0 = qblk * QB + wave * QW;
  const int qi = min(q0 + c, o.n - 1);
  const int limit = min(past + qi + 1, total); // keys this lane's query sees
  const int64_t head = ((int64_t)o.b * p.Nkv + hk) * p.Smax;
  const uint8_t* const kq = CACHE ? p.kq + head * (16 * NJ) : nullptr;
  const uint8_t* const vq = CACHE ? p.vq + head * (16 * NJ) : nullptr;
  const uint8_t* const ks = CACHE ? p.ks + head * NJ : nullptr;
  const uint8_t* const vs = CACHE ? p.vs + head * NJ : nullptr;
  const uint16_t* const kr = CACHE ? nullptr : p.k + (int64_t)o.start * p.k_ld + hk * H;
  const uint16_t* const vr = CACHE ? nullptr : p.v + (int64_t)o.start * p.v_ld + hk * H;
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

  // Item i of thread tid: 16 bytes of a row of K (V false) or of V; rows past the keys: zeros.  They pass through registers, asked
  // for D tiles before they go to LDS: two over the cache (2048 tokens behind 2048 132 -> 124 us), one for bf16 rows, whose second
  // tile would take 32 registers (1000 tokens 28.0 -> 28.9).
  i32x4 k_item[D][NC], v_item[D][NC];
  uint32_t k_byte[D][CACHE ? NC : 1], v_byte[D][CACHE ? NC : 1];
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
    if constexpr (CACHE) {
      const auto codes = rsrc((V ? vq : kq) + (int64_t)kb * (64 * 16 * NJ), rows * (16 * NJ));
      const auto scales = rsrc((V ? vs : ks) + (int64_t)kb * (64 * NJ), rows * NJ);
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const int at = i * TH + tid;
        item[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, at * 16, 0, 0));
        byte[i] = __builtin_amdgcn_raw_buffer_load_b8(scales, at, 0, 0);
      }
    } else {
      const int64_t ld = V ? p.v_ld : p.k_ld;
      const auto src = rsrc((V ? vr : kr) + (int64_t)kb * 64 * ld, rows ? (uint32_t)(((rows - 1) * (uint32_t)ld + H) * 2) : 0u);
#pragma unroll
      for (int i = 0; i < NC; i++) {
        const int at = i * TH + tid;
        item[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, (at / PER) * ((uint32_t)ld * 2) + (at % PER) * 16, 0, 0));
      }
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
      if constexpr (CACHE) {
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
      } else {
        if (partial) {
          bool some = false;
#pragma unroll
          for (int j = 0; j < 4; j++)
            some |= mx4_non_finite((uint32_t)item[i][j]);
          if (some) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              item[i][j] = (int)mx4_finite((uint32_t)item[i][j]);
          }
          odd |= some;
        }
        if (ITEMS % TH == 0 || at < ITEMS)
          *reinterpret_cast<i32x4*>(st + row * PITCH + ch * 16) = item[i];
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
  if constexpr (D == 2) {
    request(K_, ODD, 1);
    request(V_, ODD, 1);
  }
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
      // The sums are relative to a maximum that follows the true one once that is 2^8 above it (the probabilities are then at most
      // 2^8: their rounding is relative, and fp32 sums have the room).  Followed at once, nearly every tile rescales: 4 prompts of up to
      // 4100 206 us instead of 190.  What it costs is that the largest probability is no longer exactly 1: relative error against 64
      // bits 2.0e-3 there, 1.8e-3 followed at once, 1.65e-3 the rounding of the output alone.
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
        for (int i = 0; i < NV; i += 2) { // (the sum is that of the rounded ones: where a key outweighs the others its rounding cancels)
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
    if (__builtin_expect(odd_values != 0, 0)) { // (a lane reads what it wrote itself)
      const int from = mrow ? 0 : first_limit / 64 * 64;
#pragma unroll 1
      for (int d = 0; d < H; d += 4 * HALF) {
        uint16_t* const o4 = orow + d + 4 * h;
        float f[4];
        for (int e = 0; e < 4; e++)
          f[e] = bf16_bits_to_f32(o4[e]);
#pragma unroll 1
        for (int key = from; key < limit; key++) {
          if (mrow && key < p.mask_ld && bf16_bits_to_f32(mrow[key]) == -INFINITY)
            continue;
          for (int e = 0; e < 4; e++) {
            uint32_t w;
            if constexpr (CACHE)
              w = vs[(int64_t)key * NJ + (d >> 5)] == 255 ? 0x7fc0u : 0u;
            else
              w = vr[(int64_t)key * p.v_ld + d + 4 * h + e];
            if ((w & 0x7f80u) == 0x7f80u)
              f[e] += bf16_bits_to_f32(w);
          }
        }
        for (int e = 0; e < 4; e++)
          o4[e] = (uint16_t)f32_to_bf16_bits(f[e]);
      }
    }
  }
}

int mx4_prompt_launch(const char* who, const Mx4AttnParams& p, int H, bool cache, hipStream_t stream) {
  // every sequence's last workgroup may be short: at most this many, those past the last one end at once
  auto blocks = [&](int rows) { return ((int64_t)p.T + (int64_t)p.B * (rows - 1)) / rows * p.Nq; };
  const int queries = env_int("TPPX_MX4_PROMPT_QUERIES", blocks(128) >= (cache || H > 128 ? 200 : 400) ? 128 : 64);
  hipError_t e = hipSuccess;
  int rc = TPPX_OK;
  mx4_for_head(H, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    auto go = [&](auto qw, auto qg, auto kt, auto c) {
      constexpr int QW = decltype(qw)::value, QG = decltype(qg)::value, KT = decltype(kt)::value;
      auto kern = mx4_prompt_kernel<NJ, QW, QG, KT, decltype(c)::value>;
      const int64_t wgs = blocks(QW * QG);
      const size_t stages = 2 * 64 * (size_t)(mx4_k_pitch(NJ) + mx4_v_pitch(NJ, QW)), teams = KT > 1 ? QG * 64 * 16 * (size_t)(4 * NJ + 1) : 0;
      const size_t lds = std::max(stages, teams); // (the state of a second team)
      if (wgs >= ((int64_t)1 << 31)) {
        rc = set_error(TPPX_ESHAPE, "%s: problem too large", who);
        return;
      }
      e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds);
      if (e == hipSuccess)
        kern<<<dim3((unsigned)wgs), dim3(QG * KT * 64), lds, stream>>>(p);
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    constexpr std::integral_constant<int, 8> eight{};
    constexpr std::integral_constant<int, 16> q16{};
    constexpr std::integral_constant<int, 32> q32{};
    auto with_source = [&](auto qw, auto qg, auto kt) {
      if (cache)
        go(qw, qg, kt, std::true_type{});
      else
        go(qw, qg, kt, std::false_type{});
    };
    if constexpr (NJ > 4) {
      // 192 and 256 wide: one workgroup's tiles fill the LDS of a CU, and 32 queries a wave its registers at one wave per SIMD; with 16
      // queries two fit (2048 tokens x 16 heads of 256: 94.7 us, four waves of 32 queries 118; four waves of 16 112).  Few: 500 tokens
      // behind 700, 64 workgroups of 128 queries: 58.9, of 64: 51.7.
      if (queries >= 128)
        with_source(q16, eight, one);
      else
        with_source(q16, four, one);
    } else {
      // 128 queries in four waves, two workgroups on a CU, from 400 of them on (2048 tokens x 32 heads, 512: 63.7 us, the others 70.7 and
      // 68.1; 4 prompts of up to 4100 186, 220 and 241; 32-wide waves in eight 128-register ones of 16 queries 59.7 and 210).  Below that
      // two teams halve the way through a tile: over the cache four groups of queries share an expanded tile from 200 on (512 tokens x
      // 64 heads behind 6000 keys, 256: 134, 153 with two groups and 167 with one team; 64 tokens behind 4000, 64: 82 and 85), otherwise two
      // groups (1000 tokens x 32 heads, 256: 28.0, four 28.3, one team 32.8; 333 tokens 12.7, 14.5 and 15.4).
      if (queries >= 128 && (!cache || blocks(128) >= 400))
        with_source(q32, four, one);
      else if (queries >= 128)
        go(q32, four, two, std::true_type{});
      else
        with_source(q32, two, two);
    }
  });
  if (rc)
    return rc;
  if (e != hipSuccess)
    return check_hip(e, who);
  return check_hip(hipGetLastError(), who);
}
} // namespace tppx
