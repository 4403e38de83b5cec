// Attention of prompts, causal, over packed bf16 rows or over the MXFP4 cache.
#include "tppx_mx4.h"

namespace tppx {

// ---------------------------------------------------------------------------
// Prompts: QG groups of 32 queries of one head, each a wave, or with KT = 2 two that take half of every tile's keys (and are
// merged at the end: launches of few workgroups), share K and V tiles of 64 keys, bf16 in LDS in two stages, from packed rows or
// from the cache (its codes expanded once per workgroup on the way to LDS).  Both products run transposed on the 32 x 32 x 16
// MFMA: scores^T[key][query] = K Q^T, out^T[channel][query] += V^T P^T; a lane holds 16 keys of one query in the score tile, and
// those, rounded to bf16, are the second operand of the V product as they lie; V's operand is read by the transposing LDS read.
// 32 queries per wave: an operand read from LDS feeds 32 columns, with 16 the LDS (128 bytes per cycle) would take twice the
// MFMAs' time.  Scores in fp32, running maximum and sum per query.
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
constexpr int mx4_k_pitch(int NJ) { return 64 * NJ + 16; }
constexpr int mx4_v_pitch(int NJ) { return NJ % 4 == 3 ? 64 * NJ : 64 * NJ + 64; }

template <int NJ, int QG, int KT, bool CACHE>
__global__ void __launch_bounds__(QG * KT * 64, NJ <= 4 ? 2 : 1)
mx4_prompt_kernel(const Mx4AttnParams p) {
  constexpr int H = 32 * NJ, KP = mx4_k_pitch(NJ), VP = mx4_v_pitch(NJ), STAGE = 64 * (KP + VP); // K rows, then V rows
  constexpr int QB = 32 * QG, TH = 64 * QG * KT, NT = 2 / KT; // runs of 32 keys of a tile that a wave takes
  constexpr int PER = CACHE ? NJ : 4 * NJ, ITEMS = 64 * PER, NC = (ITEMS + TH - 1) / TH; // items of a row, of a tile, of a thread
  extern __shared__ __align__(16) uint8_t lds[]; // 2 stages
  __shared__ int odd_values;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % QG, team = __builtin_amdgcn_readfirstlane(tid >> 6) / QG;
  const int c = lane & 31, h = lane >> 5;
  // heads go round the XCDs, those of one K/V head to the same one
  const int hr = (int)blockIdx.x % p.Nq, hk = hr % p.Nkv, hq = hk * p.R + hr / p.Nkv;
  Block o;
  if (!locate(p.cu, p.B, p.T, 1, QB, (int)blockIdx.x / p.Nq, o))
    return;
  const int qblk = (o.n + QB - 1) / QB - 1 - o.at; // the last queries see the most keys: first
  const int past = CACHE ? max(p.past[o.b], 0) : 0;
  const int total = CACHE ? min(past + o.n, p.Smax) : o.n; // keys of the sequence
  const int q0 = qblk * QB + wave * 32;
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

  bf16x8 q[2 * NJ];
  {
    const uint16_t* qrow = p.q + (int64_t)(o.start + qi) * p.q_ld + (int64_t)hq * H + h * 8;
#pragma unroll
    for (int j = 0; j < 2 * NJ; j++)
      q[j] = *reinterpret_cast<const bf16x8*>(qrow + j * 16);
  }
  // keys that some query of this workgroup sees
  const int keys = min(past + min(qblk * QB + QB, o.n), total), tiles = (keys + 63) / 64;
  const int first_limit = min(past + qblk * QB + 1, total); // keys that all of them see

  // Item i of thread tid: 16 bytes of a row of K (V false) or of V; rows past the keys: zeros.  They pass through registers, asked
  // for a whole tile before they go to LDS.
  i32x4 k_item[NC], v_item[NC];
  uint32_t k_byte[CACHE ? NC : 1], v_byte[CACHE ? NC : 1];
  // (buffers of a tile's rows: what lies past them reads as zero, with no branch and no access)
  auto request = [&](auto V_, int kb) {
    constexpr bool V = decltype(V_)::value;
    auto& item = V ? v_item : k_item;
    auto& byte = V ? v_byte : k_byte;
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
  auto deliver = [&](auto V_, int kb, int stage) {
    constexpr bool V = decltype(V_)::value;
    auto& item = V ? v_item : k_item;
    auto& byte = V ? v_byte : k_byte;
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
            *reinterpret_cast<bf16x8*>(dst + (V ? (j ^ (row & 3)) * 16 : j * 16)) =
                mx4_to_bf16(nan ? 0u : (uint32_t)(V ? chunk_of(item[i], j ^ (row & 3)) : item[i][j]), s); // (zero times infinity)
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
        *reinterpret_cast<i32x4*>(st + row * PITCH + ch * 16) = item[i];
      }
    }
    if (odd)
      odd_values = 1;
  };
  constexpr std::false_type K_{};
  constexpr std::true_type V_{};

  float m = LOWEST, l = 0.f;
  f32x16 acc[NJ];
#pragma unroll
  for (int dt = 0; dt < NJ; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++)
      acc[dt][i] = 0.f;
  const float scale2 = p.scale * LOG2E;
  const int wave_limit = min(past + min(q0 + 32, o.n), total); // keys that some query of this wave sees
  const bool idle = q0 >= o.n;

  if (tid == 0)
    odd_values = 0;
  request(K_, 0);
  request(V_, 0);
  __syncthreads();
  deliver(K_, 0, 0);
  request(K_, 1);
  deliver(V_, 0, 0);
  request(V_, 1);
  for (int kb = 0; kb < tiles; kb++) {
    const int stage = kb & 1;
    __syncthreads(); // this tile has been written, the other stage has been read
    const bool more = kb + 1 < tiles, busy = !idle && kb * 64 < wave_limit; // (uniform in a wave)
    const uint8_t* const st = lds + stage * STAGE;
    bf16x8 pb[2 * NT];
    if (busy) {
      f32x16 sc[NT];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < 16; i++)
          sc[t][i] = 0.f;
#pragma unroll
        for (int j = 0; j < 2 * NJ; j++)
          sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(st + ((team + t) * 32 + c) * KP + j * 32 + h * 16), q[j], sc[t], 0, 0, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      // key of score i of run t
      auto key_of = [&](int t, int i) { return kb * 64 + (team + t) * 32 + (i & 3) + 8 * (i >> 2) + 4 * h; };
      if (mrow) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
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
          for (int i = 0; i < 16; i++)
            sc[t][i] = key_of(t, i) < limit ? sc[t][i] : -INFINITY;
      }
      float mx = m;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          mx = fmaxf(mx, sc[t][i]);
      const float unit = mrow ? LOG2E : scale2;
      float alpha = 1.f;
      // The sums are relative to a maximum that follows the true one once that is 2^8 above it (the probabilities are then at most
      // 2^8: their rounding is relative, and fp32 sums have the room); followed at once, nearly every tile would rescale.
      if (__builtin_amdgcn_ballot_w64((mx - m) * unit > 8.f) != 0) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        alpha = __builtin_amdgcn_exp2f((m - mx) * unit);
#pragma unroll
        for (int dt = 0; dt < NJ; dt++)
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
        for (int i = 0; i < 16; i++) {
          const float pr = __builtin_amdgcn_exp2f(fmaf(sc[t][i], unit, off));
          l += pr;
          pb[t * 2 + (i >> 3)][i & 7] = (__bf16)pr;
        }
    }
    if (more) {
      deliver(K_, kb + 1, stage ^ 1);
      request(K_, kb + 2);
    }
    if (busy) {
      // V operand of 16 keys (step u) and 32 channels: two transposing reads of 4 keys each for this lane's half
      const uint8_t* const vt = st + 64 * KP + (team * 32 + 4 * h + ((lane & 15) >> 2)) * VP + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
      auto operand = [&](int dt, int u, int e) {
        return __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(vt + (u * 16 + e * 8) * VP + dt * 64)));
      };
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < 2 * NT; u++)
#pragma unroll
        for (int dt = 0; dt < NJ; dt++) {
          const i32x2 a = operand(dt, u, 0), b = operand(dt, u, 1);
          const i32x4 w = {a[0], a[1], b[0], b[1]};
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), pb[u], acc[dt], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (more) {
      deliver(V_, kb + 1, stage ^ 1);
      request(V_, kb + 2);
    }
  }
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
    for (int dt = 0; dt < NJ; dt++)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint2 w = make_uint2(f32x2_to_bf16_bits(acc[dt][i] * inv, acc[dt][i + 1] * inv), f32x2_to_bf16_bits(acc[dt][i + 2] * inv, acc[dt][i + 3] * inv));
        *reinterpret_cast<uint2*>(orow + dt * 32 + 8 * (i >> 2) + 4 * h) = w;
      }
    if (__builtin_expect(odd_values != 0, 0)) { // (a lane reads what it wrote itself)
      const int from = mrow ? 0 : first_limit / 64 * 64;
#pragma unroll 1
      for (int d = 0; d < H; d += 8) {
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
  const bool wide = blocks(128) >= 400;
  const int64_t wgs = wide ? blocks(128) : blocks(64);
  TPPX_REQUIRE(wgs < ((int64_t)1 << 31), TPPX_ESHAPE, "%s: problem too large", who);
  hipError_t e = hipSuccess;
  mx4_for_head(H, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    auto go = [&](auto qg, auto c) {
      constexpr int QG = decltype(qg)::value;
      auto kern = mx4_prompt_kernel<NJ, QG, 4 / QG, decltype(c)::value>;
      const size_t lds = 2 * 64 * (size_t)(mx4_k_pitch(NJ) + mx4_v_pitch(NJ));
      e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds);
      if (e == hipSuccess)
        kern<<<dim3((unsigned)wgs), dim3(256), lds, stream>>>(p);
    };
    auto with_source = [&](auto qg) {
      if (cache)
        go(qg, std::true_type{});
      else
        go(qg, std::false_type{});
    };
    if (wide)
      with_source(std::integral_constant<int, 4>{});
    else
      with_source(std::integral_constant<int, 2>{});
  });
  if (e != hipSuccess)
    return check_hip(e, who);
  return check_hip(hipGetLastError(), who);
}

} // namespace tppx
