// Key/value cache in pages, bf16, for sequences of different lengths, and passes that check drafted tokens over it: norm, rotation
// and append to the pages, attention of single tokens, of trees of drafted tokens and of pieces of prompts, and the move of the
// accepted tokens' keys.
//
// A layer: [2][pages][Nkv][page][H], keys then values; slot s of sequence b lies in page table[b][s / page] at s % page.  The tokens of
// a step ("nodes") are packed: sequence b owns rows cu[b] .. cu[b + 1] - 1 and held past[b] keys before them; cu null: one each.  Node i
// goes to slot past + i.  parents[i] is the node of the same sequence that node i continues; without parents that is node i - 1.  All of
// these arrays live on the device and are clamped there, so that no value in them leads out of a buffer.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "tppx_mx4.h"

namespace tppx {

// ---------------------------------------------------------------------------
// shared by the kernels
// ---------------------------------------------------------------------------
struct Pages {
  const int32_t* table; // [B][table_ld]
  int64_t table_ld;     // pages of a sequence
  int pages, shift;     // of a layer; log2 of a page's slots
};
// The page of slot `s` of sequence b, or -1: none.
__device__ __forceinline__ int page_of(const Pages& g, int b, int s) {
  const int i = s >> g.shift;
  if (s < 0 || i >= g.table_ld)
    return -1;
  const int id = g.table[(int64_t)b * g.table_ld + i];
  return (unsigned)id < (unsigned)g.pages ? id : -1;
}
// element offset of a head's slot `at` in a page of one side of a layer
__device__ __forceinline__ int64_t slot_at(const Pages& g, int id, int Nkv, int head, int at, int H) {
  return ((((int64_t)id * Nkv + head) << g.shift) + (at & ((1 << g.shift) - 1))) * H;
}
// the node that node i of a sequence continues, or -1 (also for what is no earlier node)
__device__ __forceinline__ int parent_of(const int32_t* parents, int i) {
  const int j = parents ? parents[i] : i - 1;
  return j < i ? max(j, -1) : -1;
}
// Sequence of a packed row, its first row and length; false: the row belongs to none.
__device__ __forceinline__ bool sequence_at(const int32_t* cu, int B, int T, int row, int& b, int& first, int& n) {
  b = first = row;
  n = 1;
  if (!cu)
    return row < B;
  b = sequence_of(cu, B, __builtin_amdgcn_readfirstlane(row)); // of the wave's first row
  while (b < B && cu[b + 1] <= row)
    b++;
  if (b >= B || row < cu[0])
    return false;
  first = cu[b];
  n = min(cu[b + 1], T) - first;
  return first >= 0 && first <= row;
}

// ---------------------------------------------------------------------------
// Norm, rotation and append, as the MXFP4 cache's: a thread keeps its token, the heads go by.  Everything in fp32, one rounding.  A node's
// position, where none is given, is past + the number of nodes that it continues.
// ---------------------------------------------------------------------------
struct PagedRowsParams {
  const uint16_t *q, *k, *v; // [T][heads][H], rows *_ld elements apart; q may be null
  uint16_t *qo, *layer;
  const void *gq, *gk;       // [H] f32 or bf16, or null
  const float* emb;          // [2][MP][HR] cos / sin, or with gptj [MP][HR] sin | cos, or null
  const int64_t* pos;        // [T], or null
  const int32_t *past, *cu, *parents;
  Pages g;
  int64_t q_ld, k_ld, v_ld;
  int T, B, Nq, Nkv, H, MP, HR;
  int gptj, gamma_f32;
  float eps;
};

template <int G>
__global__ void __launch_bounds__(256)
paged_rows_kernel(const PagedRowsParams p) {
  constexpr int TB = 256 / G; // tokens of a workgroup
  const int u = threadIdx.x % G, mine = (int)blockIdx.x * TB + (int)threadIdx.x / G, tok = min(mine, p.T - 1);
  const int nq = p.q ? p.Nq : 0, nk = p.Nkv, total = nq + 2 * nk;
  Mx4Lane t;
  mx4_share<G>(p, u, t);
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
  int b, first, n;
  const bool here = sequence_at(p.cu, p.B, p.T, tok, b, first, n) && mine < p.T;
  b = min(b, p.B - 1);
  const int past = p.past[b], node = tok - first;
  const int64_t slot = (int64_t)past + node;
  int64_t at = slot;
  if (p.pos) {
    at = p.pos[tok];
  } else if (p.parents && here) {
    int depth = 0;
    for (int j = parent_of(p.parents + first, node); j >= 0; j = parent_of(p.parents + first, j))
      depth++;
    at = (int64_t)past + depth;
  }
  const int page = past >= 0 && slot < ((int64_t)1 << 30) && here ? page_of(p.g, b, (int)slot) : -1;
  mx4_angles(p, u, at, t);
  uint4 w[2];
  auto step = [&]() {
    w[0] = next[0];
    w[1] = next[1];
    if (!t.live) // (heads of 96 and 192 leave lanes over)
      w[0] = w[1] = make_uint4(0, 0, 0, 0);
    load(row + (int)gridDim.y);
  };
  auto write = [&](uint16_t* to, const uint4& a, const uint4& z) {
    uint4* const dst = reinterpret_cast<uint4*>(to);
    dst[t.c[0]] = a;
    dst[t.c[1]] = z;
  };
  for (; row < nq; row += (int)gridDim.y) {
    step();
    float y[2][8];
    mx4_turn<G>(p, w, t, p.gq, y);
    if (t.live && here)
      write(p.qo + ((int64_t)tok * p.Nq + row) * p.H, pack8(y[0]), pack8(y[1]));
  }
  for (; row < nq + nk; row += (int)gridDim.y) {
    step();
    float y[2][8];
    mx4_turn<G>(p, w, t, p.gk, y);
    if (t.live && page >= 0)
      write(p.layer + slot_at(p.g, page, p.Nkv, row - nq, (int)slot, p.H), pack8(y[0]), pack8(y[1]));
  }
  const int64_t values = (((int64_t)p.g.pages * p.Nkv) << p.g.shift) * p.H;
  for (; row < total; row += (int)gridDim.y) {
    step();
    if (t.live && page >= 0)
      write(p.layer + values + slot_at(p.g, page, p.Nkv, row - nq - nk, (int)slot, p.H), w[0], w[1]);
  }
}

// ---------------------------------------------------------------------------
// Attention: a workgroup for a node's query head, a wave takes 64 keys at a time.
// ---------------------------------------------------------------------------
struct PagedAttnParams {
  const uint16_t *q, *layer;
  const int32_t *past, *cu, *parents;
  uint16_t* out; // [T][Nq][H]
  Pages g;
  int64_t q_ld;
  int T, B, Nq, Nkv, H;
  float scale;
};

__global__ void __launch_bounds__(256)
paged_attn_kernel(const PagedAttnParams p) {
  __shared__ float q[256], part[4][256], stat[4][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = (int)blockIdx.x, hq = (int)blockIdx.y, hk = hq / (p.Nq / p.Nkv);
  int b, first, n;
  if (!sequence_at(p.cu, p.B, p.T, row, b, first, n))
    return;
  const int node = row - first, past = p.past[b];
  const int capacity = (int)min(p.g.table_ld << p.g.shift, (int64_t)1 << 30);
  const int keys = past < 0 ? 0 : (int)min((int64_t)past + node + 1, (int64_t)capacity);
  const int32_t* const parents = p.parents ? p.parents + first : nullptr;
  if (tid < p.H)
    q[tid] = bf16_bits_to_f32(p.q[(int64_t)row * p.q_ld + (int64_t)hq * p.H + tid]) * p.scale;
  __syncthreads();
  const int64_t values = (((int64_t)p.g.pages * p.Nkv) << p.g.shift) * p.H;
  float m = LOWEST, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * 64; k0 < keys; k0 += 256) {
    const int key = k0 + lane;
    bool seen = key < keys;
    if (seen && key >= past && parents) {
      int j = node;
      while (j > key - past)
        j = parent_of(parents, j);
      seen = j == key - past;
    }
    const int id = seen ? page_of(p.g, b, key) : -1;
    const int64_t at = id >= 0 ? slot_at(p.g, id, p.Nkv, hk, key, p.H) : -1;
    float s = -INFINITY;
    if (at >= 0) {
      s = 0.f;
      for (int d = 0; d < p.H; d++)
        s = fmaf(q[d], bf16_bits_to_f32(p.layer[at + d]), s);
    }
    float mx = fmaxf(m, s);
    for (int d = 1; d < 64; d *= 2)
      mx = fmaxf(mx, __shfl_xor(mx, d));
    const float alpha = expf(m - mx), e = at >= 0 ? expf(s - mx) : 0.f;
    m = mx;
    l = l * alpha + e;
    for (int i = 0; i < 4; i++)
      acc[i] *= alpha;
    for (int j = 0; j < 64; j++) {
      const int64_t from = __shfl(at, j);
      const float pj = __shfl(e, j);
      if (from >= 0)
        for (int i = 0; i * 64 + lane < p.H; i++)
          acc[i] = fmaf(pj, bf16_bits_to_f32(p.layer[values + from + i * 64 + lane]), acc[i]);
    }
  }
  for (int d = 1; d < 64; d *= 2)
    l += __shfl_xor(l, d);
  for (int i = 0; i < 4; i++)
    part[wave][i * 64 + lane] = acc[i];
  if (lane == 0) {
    stat[wave][0] = m;
    stat[wave][1] = l;
  }
  __syncthreads();
  if (tid < p.H) {
    float mx = LOWEST, sum = 0.f, v = 0.f;
    for (int w = 0; w < 4; w++)
      mx = fmaxf(mx, stat[w][0]);
    for (int w = 0; w < 4; w++) {
      const float a = expf(stat[w][0] - mx);
      sum = fmaf(a, stat[w][1], sum);
      v = fmaf(a, part[w][tid], v);
    }
    p.out[((int64_t)row * p.Nq + hq) * p.H + tid] = (uint16_t)f32_to_bf16_bits(sum != 0.f ? v / sum : 0.f);
  }
}

// ---------------------------------------------------------------------------
// The keys and values of an accepted path to the slots from past on, in all layers.  A thread takes 16 bytes of a head's row through the
// whole path: node path[i] goes to slot past + i, and as path ascends no row is read after another was written over it.
// ---------------------------------------------------------------------------
struct PagedKeepParams {
  uint16_t* cache; // [sides][pages][Nkv][page][H], sides = 2 layers
  const int32_t *past, *path, *count, *cu;
  Pages g;
  int T, B, Nkv, H, sides;
};

__global__ void __launch_bounds__(256)
paged_keep_kernel(const PagedKeepParams p) {
  const int b = (int)blockIdx.x, per = p.H / 8, items = p.Nkv * per;
  const int64_t item = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (item >= (int64_t)items * p.sides)
    return;
  const int side = (int)(item / items), in = (int)(item % items), head = in / per, ch = in % per;
  const int first = p.cu ? p.cu[b] : b, n = p.cu ? min(p.cu[b + 1], p.T) - first : 1;
  const int past = p.past[b];
  if (first < 0 || n < 1 || past < 0 || past > (1 << 30))
    return;
  const int count = min(p.count[b], n);
  uint16_t* const at = p.cache + (int64_t)side * ((((int64_t)p.g.pages * p.Nkv) << p.g.shift) * p.H) + ch * 8;
  for (int i = 0; i < count; i++) {
    const int from = p.path[first + i];
    if (from <= i || from >= n) // (in its place already, or no node)
      continue;
    const int a = page_of(p.g, b, past + from), z = page_of(p.g, b, past + i);
    if (a >= 0 && z >= 0)
      *reinterpret_cast<uint4*>(at + slot_at(p.g, z, p.Nkv, head, past + i, p.H)) = *reinterpret_cast<const uint4*>(at + slot_at(p.g, a, p.Nkv, head, past + from, p.H));
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int paged_checks(const char* who, const void* table, const void* past, const void* cu, int64_t T, int64_t B, int64_t Nkv, int64_t H,
                        int64_t pages, int64_t page, int64_t table_ld, Pages& g) {
  TPPX_REQUIRE(table && past, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE((((uintptr_t)table | (uintptr_t)past | (uintptr_t)cu) & 3u) == 0, TPPX_EINVAL, "%s: pointer not 4-byte aligned", who);
  TPPX_REQUIRE(mx4_has_head(H), TPPX_EUNSUPPORTED, "%s: head size %ld (64, 96, 128, 192 and 256 are built)", who, (long)H);
  TPPX_REQUIRE(page >= 16 && page <= (1 << 16) && (page & (page - 1)) == 0, TPPX_EUNSUPPORTED, "%s: pages of %ld slots (powers of two from 16 to 65536 are built)", who, (long)page);
  TPPX_REQUIRE(T >= 0 && T < ((int64_t)1 << 30) && B > 0 && B < ((int64_t)1 << 24) && Nkv > 0 && Nkv <= (1 << 16), TPPX_ESHAPE,
               "%s: bad shape T=%ld B=%ld Nkv=%ld", who, (long)T, (long)B, (long)Nkv);
  TPPX_REQUIRE(pages > 0 && pages < ((int64_t)1 << 31) && table_ld > 0 && table_ld * page <= ((int64_t)1 << 30), TPPX_ESHAPE,
               "%s: %ld pages, %ld of a sequence", who, (long)pages, (long)table_ld);
  TPPX_REQUIRE(cu || T == B, TPPX_ESHAPE, "%s: %ld tokens of %ld sequences need their bounds", who, (long)T, (long)B);
  g.table = (const int32_t*)table;
  g.table_ld = table_ld;
  g.pages = (int)pages;
  g.shift = __builtin_ctzll((unsigned long long)page);
  return TPPX_OK;
}

} // namespace tppx

using namespace tppx;

extern "C" int tppx_append_paged(const void* q, const void* k, const void* v, const void* gamma_q, const void* gamma_k, int gamma_dtype,
                                 float eps, const void* emb_pos, int gptj, const void* pos, void* layer, const void* table, const void* past,
                                 const void* cu, const void* parents, void* q_out, int64_t T, int64_t B, int64_t Nq, int64_t Nkv, int64_t H,
                                 int64_t pages, int64_t page, int64_t table_ld, int64_t q_ld, int64_t k_ld, int64_t v_ld, int64_t MP,
                                 int64_t HR, tppx_stream_t stream) {
  const char* who = "tppx_append_paged";
  TPPX_REQUIRE(k && v && layer && (!q || q_out), TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(layer) && aligned16(gamma_q) && aligned16(gamma_k) && aligned16(emb_pos),
               TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  TPPX_REQUIRE(((uintptr_t)parents & 3u) == 0 && ((uintptr_t)pos & 7u) == 0, TPPX_EINVAL, "%s: parents or positions not aligned", who);
  TPPX_REQUIRE(gamma_dtype == TPPX_DT_F32 || gamma_dtype == TPPX_DT_BF16, TPPX_EINVAL, "%s: gamma dtype %d", who, gamma_dtype);
  PagedRowsParams p;
  memset(&p, 0, sizeof(p));
  if (int rc = paged_checks(who, table, past, cu, T, B, Nkv, H, pages, page, table_ld, p.g))
    return rc;
  TPPX_REQUIRE(!q || (Nq > 0 && Nq <= (1 << 16)), TPPX_ESHAPE, "%s: Nq=%ld", who, (long)Nq);
  TPPX_REQUIRE(!emb_pos || (MP > 0 && MP < ((int64_t)1 << 31) && HR > 0 && HR <= H && HR % 16 == 0), TPPX_ESHAPE,
               "%s: rotary_dim=%ld must be a multiple of 16 and <= H=%ld", who, (long)HR, (long)H);
  TPPX_REQUIRE((!q || q_ld >= Nq * H) && k_ld >= Nkv * H && v_ld >= Nkv * H && ((q ? q_ld : 0) | k_ld | v_ld) % 8 == 0, TPPX_ESHAPE,
               "%s: row strides must be multiples of 8 elements and hold a row", who);
  if (T == 0)
    return TPPX_OK;
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k; p.v = (const uint16_t*)v; p.qo = (uint16_t*)q_out; p.layer = (uint16_t*)layer;
  p.gq = gamma_q; p.gk = gamma_k; p.gamma_f32 = gamma_dtype == TPPX_DT_F32; p.eps = eps;
  p.emb = (const float*)emb_pos; p.gptj = gptj != 0; p.pos = (const int64_t*)pos;
  p.past = (const int32_t*)past; p.cu = (const int32_t*)cu; p.parents = (const int32_t*)parents;
  p.q_ld = q ? q_ld : 0; p.k_ld = k_ld; p.v_ld = v_ld;
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.H = (int)H; p.MP = (int)MP; p.HR = emb_pos ? (int)HR : 0;
  const int G = H <= 64 ? 4 : H <= 128 ? 8 : 16;
  const int64_t rows = (q ? Nq : 0) + 2 * Nkv, blocks = (T * G + 255) / 256;
  const int64_t per_block = std::max<int64_t>(1, std::min<int64_t>({rows, 65535, 1024 / blocks}));
  const dim3 grid((unsigned)blocks, (unsigned)per_block);
  if (G == 4)
    paged_rows_kernel<4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p);
  else if (G == 8)
    paged_rows_kernel<8><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p);
  else
    paged_rows_kernel<16><<<grid, dim3(256), 0, (hipStream_t)stream>>>(p);
  return check_hip(hipGetLastError(), who);
}

extern "C" int tppx_attn_paged(const void* q, const void* layer, const void* table, const void* past, const void* cu, const void* parents,
                               void* out, int64_t T, int64_t B, int64_t Nq, int64_t Nkv, int64_t H, int64_t pages, int64_t page,
                               int64_t table_ld, int64_t q_ld, void* ws, int64_t ws_bytes, void* counters, int64_t counter_bytes,
                               tppx_stream_t stream) {
  const char* who = "tppx_attn_paged";
  TPPX_REQUIRE(q && layer && out, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(q) && aligned16(layer) && aligned16(out) && aligned16(ws), TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  TPPX_REQUIRE((((uintptr_t)parents | (uintptr_t)counters) & 3u) == 0, TPPX_EINVAL, "%s: parents or counters not 4-byte aligned", who);
  PagedAttnParams p;
  memset(&p, 0, sizeof(p));
  if (int rc = paged_checks(who, table, past, cu, T, B, Nkv, H, pages, page, table_ld, p.g))
    return rc;
  TPPX_REQUIRE(Nq > 0 && Nq <= (1 << 16) && Nq % Nkv == 0 && T * (Nq / Nkv) < ((int64_t)1 << 31), TPPX_ESHAPE, "%s: Nq=%ld, Nkv=%ld", who, (long)Nq, (long)Nkv);
  TPPX_REQUIRE(q_ld >= Nq * H && q_ld % 8 == 0, TPPX_ESHAPE, "%s: row strides must be multiples of 8 elements and hold a row", who);
  TPPX_REQUIRE(ws_bytes >= 0 && (ws_bytes == 0 || ws) && counter_bytes >= 0 && (counter_bytes == 0 || counters), TPPX_EINVAL,
               "%s: size given with a null pointer", who);
  if (T == 0)
    return TPPX_OK;
  p.q = (const uint16_t*)q; p.q_ld = q_ld; p.layer = (const uint16_t*)layer; p.out = (uint16_t*)out;
  p.past = (const int32_t*)past; p.cu = (const int32_t*)cu; p.parents = (const int32_t*)parents;
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.H = (int)H;
  p.scale = 1.0f / sqrtf((float)H);
  paged_attn_kernel<<<dim3((unsigned)T, (unsigned)Nq), dim3(256), 0, (hipStream_t)stream>>>(p);
  return check_hip(hipGetLastError(), who);
}

extern "C" int tppx_keep_paged(void* cache, const void* table, const void* past, const void* path, const void* count, const void* cu,
                               int64_t layers, int64_t T, int64_t B, int64_t Nkv, int64_t H, int64_t pages, int64_t page, int64_t table_ld,
                               tppx_stream_t stream) {
  const char* who = "tppx_keep_paged";
  TPPX_REQUIRE(cache && path && count, TPPX_EINVAL, "%s: null pointer", who);
  TPPX_REQUIRE(aligned16(cache), TPPX_EINVAL, "%s: pointer not 16-byte aligned", who);
  TPPX_REQUIRE((((uintptr_t)path | (uintptr_t)count) & 3u) == 0, TPPX_EINVAL, "%s: path or count not 4-byte aligned", who);
  PagedKeepParams p;
  memset(&p, 0, sizeof(p));
  if (int rc = paged_checks(who, table, past, cu, T, B, Nkv, H, pages, page, table_ld, p.g))
    return rc;
  TPPX_REQUIRE(layers > 0 && layers <= (1 << 16), TPPX_ESHAPE, "%s: %ld layers", who, (long)layers);
  const int64_t blocks = (2 * layers * Nkv * (H / 8) + 255) / 256;
  TPPX_REQUIRE(blocks <= 65535, TPPX_ESHAPE, "%s: problem too large", who);
  if (T == 0)
    return TPPX_OK;
  p.cache = (uint16_t*)cache;
  p.past = (const int32_t*)past; p.path = (const int32_t*)path; p.count = (const int32_t*)count; p.cu = (const int32_t*)cu;
  p.T = (int)T; p.B = (int)B; p.Nkv = (int)Nkv; p.H = (int)H; p.sides = (int)(2 * layers);
  paged_keep_kernel<<<dim3((unsigned)B, (unsigned)blocks), dim3(256), 0, (hipStream_t)stream>>>(p);
  return check_hip(hipGetLastError(), who);
}
