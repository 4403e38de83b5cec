// Key/value cache in pages, bf16, for sequences of different lengths, and passes that check drafted tokens over it: norm, rotation
// and append to the pages, attention of single tokens, of trees of drafted tokens and of pieces of prompts, and the move of the
// accepted tokens' keys.
//
// A layer: [2][pages][Nkv][page][H], keys then values; slot s of sequence b lies in page table[b][s / page] at s % page.  The tokens of
// a step ("nodes") are packed: sequence b owns rows cu[b] .. cu[b + 1] - 1 and held past[b] keys before them; cu null: one each.  Node i
// goes to slot past + i.  parents[i] is the node of the same sequence that node i continues; without parents that is node i - 1.  All of
// these arrays live on the device and are clamped there, so that no value in them leads out of a buffer.
#include <limits.h>
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
// position, where none is given, is past + the number of nodes that it continues.  Copy work: 24 trees of 20 to 61 nodes, 64 + 16 heads
// of 128 (36.7 MB) 10.2 us, 3.6 TB/s; one token 3.1 us, a launch and one way to memory and back.
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
// Attention.  The columns of a sequence's K/V head are its (node, query head) pairs; a workgroup takes 16 CW of them, the columns of 16 x 16
// x 32 MFMAs, for a part of the keys.  Both products run transposed, scores^T[key][col] = K Q^T and out^T[channel][col] += V^T P^T: the
// scores of a lane are those of one column, and rounded to bf16 they are the second operand of the V product as they lie.  TW teams of
// CW waves take tiles of KEYS keys in turn, from the last one down.  A tile's rows come by loads straight into LDS, one tile ahead,
// a run of 16 rows at a time: a page holds whole runs, so its number is the same for all lanes.
// A node sees the slots before the step's and of the step's those of the nodes that it continues: in the tiles that hold such slots a
// lane follows its column's node up and sets a bit for each of the tile's keys that it meets; as tiles descend, it goes on where the
// tile above ended.
// A key that a column does not see adds nothing whatever it holds: its score is replaced, and in those tiles values that are infinite
// or NaN are added one by one to the columns that see them and become zeros in LDS.
// Scores, maxima, sums and outputs in fp32; rounded to bf16 are the probabilities (the second product's operand; their sum is taken over the
// rounded ones, so that the weights add up to one) and the result.
// What bounds it: of single tokens the cache's bytes (48 sequences of up to 9000 keys, 64 heads on 8 of 128: 752 MB in 140 us, 5.4 TB/s,
// above a large copy's 4.9).  Of long pieces of prompts the clock: 1024 tokens behind 8000 keys 282 us, 1010 TFLOP/s, at 1.8 of 2.4 GHz with
// the matrix instructions busy in half of the cycles, the others' issue in 0.4 of them, LDS in a quarter (a library product of 8192^3
// reaches 1560).  Of small steps the way through it: 8 nodes behind 50 keys 7.1 us, 60 behind 5000 (28 heads on 4) 19.5 + 4 for the merge, of
// which tiles are 7.  Not faster: the scores of the next tile under the weights of this one (registers), 64 columns a wave at one wave
// per SIMD (282 -> 361 us), s_setprio around the products.
// ---------------------------------------------------------------------------
struct PagedAttnParams {
  const uint16_t *q, *layer;
  const int32_t *past, *cu, *parents;
  uint16_t* out; // [T][Nq][H]
  float* part;   // [part][cols][H], then, behind `parts` of those, [part][cols][2], then the units to merge
  int parts;     // at most
  unsigned int* counters;
  Pages g;
  int64_t q_ld;
  int T, B, Nq, Nkv, R;
  int target, most;  // items of a launch that run at once (0: units are not split), that there may be
  int least;         // tiles of one at least
  float scale;
};
// what the merge has to know of a unit: parts (1: nothing to do), the first one's place, from one to the next, the last one's; its
// K/V head, first row, columns in front of it and in it
struct Merge {
  int S, first, stride, last, hk, start, col0, ncol;
};
// [0].S: how many follow
template <int COLS, int H>
__device__ __forceinline__ Merge* merges_of(const PagedAttnParams& p) { return reinterpret_cast<Merge*>(p.part + (int64_t)p.parts * (COLS * (H + 2))); }
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t* ConstantInts; // (scalar loads)

constexpr int MAX_SPLITS = 64;
constexpr int PAGED_NODES = 256;

// The work of a launch, laid out on the device, where the lengths are: an item is a part of a unit's keys, a unit a block of a sequence's
// columns for one K/V head.  Parts are of about `chunk` tiles: long sequences are split where short ones are not, and in all there are
// no more than run at once, or, where that leaves parts 1.4 times the mean and longer than 2048 keys, some rounds of them (30 single
// tokens behind up to 9000 keys 105 -> 93 us).  More units than run at once, none longer than 1.2 of the mean share: not split (64 of up
// to 2000 50 us, split 60).  Items of a sequence: [split][block][K/V head].
// ROUNDS: as many units as fill whole rounds of what runs at once are not split and come first, then the parts of the others: all that
// are of `chunk` tiles, of a sequence [split][block][K/V head], then the last ones, of the first keys, [block][K/V head].  If those are
// short enough a few of them run one after another beside the others (700 tokens behind 9000 keys, 352 units where 512 run: 309 us
// unsplit, 266 so).  Blocks go down, the longest first (8000 tokens without a past 1516 -> 1418 us).
// A K/V head is an item's last index: its workgroups lie on one XCD where there are eight, and share that one's L2.
struct Item {
  Block o;           // sequence, its first row and nodes, block
  int hk, S;         // of S parts
  int low, high;     // tiles
  int first, stride; // the unit's first part, from one's to the next one's
  int last, mine;    // its last part, this item's
  int unit, units;   // its place among those that may be split, where this is the last part (else -1); how many there are, all told
  __device__ __forceinline__ int part(int s) const { return s < S - 1 ? first + s * stride : last; }
};
// keys that the nodes of sequence b up to `last` see, of which that one sees most
__device__ __forceinline__ int paged_past(const PagedAttnParams& p, int b) { return min(p.past[b], (int)(p.g.table_ld << p.g.shift)); }
__device__ __forceinline__ int paged_keys(const PagedAttnParams& p, int past, int last) {
  return past < 0 ? 0 : (int)min((int64_t)past + last + 1, p.g.table_ld << p.g.shift);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_lane(int v) { // (0 where there is no such lane)
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, ROWS == 0xf);
}
// sum over the lanes below, and this one's; all lanes take part
__device__ __forceinline__ int scan_wave(int v) {
  v += from_lane<0x111, 0xf>(v); // row_shr:1
  v += from_lane<0x112, 0xf>(v);
  v += from_lane<0x114, 0xf>(v);
  v += from_lane<0x118, 0xf>(v);
  v += from_lane<0x142, 0xa>(v); // row_bcast:15 into the second and the last row
  v += from_lane<0x143, 0xc>(v); // row_bcast:31 into the upper rows
  return v;
}
__device__ __forceinline__ int sum_of_wave(int v) { return __builtin_amdgcn_readlane(scan_wave(v), 63); }
__device__ __forceinline__ int max_of_wave(int v) { // of none below 0
  v = max(v, from_lane<0x111, 0xf>(v));
  v = max(v, from_lane<0x112, 0xf>(v));
  v = max(v, from_lane<0x114, 0xf>(v));
  v = max(v, from_lane<0x118, 0xf>(v));
  v = max(v, from_lane<0x142, 0xa>(v));
  v = max(v, from_lane<0x143, 0xc>(v));
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ float sum_of_wave(float v) {
  auto add = [&](auto c, auto r) { v += __int_as_float(from_lane<decltype(c)::value, decltype(r)::value>(__float_as_int(v))); };
  constexpr std::integral_constant<int, 15> all{};
  add(std::integral_constant<int, 0x111>{}, all);
  add(std::integral_constant<int, 0x112>{}, all);
  add(std::integral_constant<int, 0x114>{}, all);
  add(std::integral_constant<int, 0x118>{}, all);
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 10>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 12>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// Item `id`; false past the last one.  All lanes of a wave take part.
template <int COLS, int KEYS, bool ROUNDS>
__device__ __forceinline__ bool locate_item(const PagedAttnParams& p, int id, Item& it) {
  const int lane = threadIdx.x & 63;
  it.hk = id % p.Nkv;
  it.units = 0;
  id /= p.Nkv;
  struct Seq {
    int s, n, blocks, past;
  };
  auto seq = [&](int b) {
    Seq q = {0, 0, 0, 0};
    if (b < p.B) {
      const int s = p.cu ? min(max(p.cu[b], 0), p.T) : b, e = p.cu ? min(max(p.cu[b + 1], 0), p.T) : b + 1;
      q.s = s;
      q.n = max(e - s, 0);
      q.blocks = (int)(((int64_t)q.n * p.R + COLS - 1) / COLS);
      q.past = paged_past(p, b);
    }
    return q;
  };
  auto tiles_of = [&](const Seq& z, int tail) { // of its first `tail` blocks, at most
    return tail ? (paged_keys(p, z.past, !ROUNDS || tail == z.blocks ? z.n - 1 : (tail * COLS - 1) / p.R) + KEYS - 1) / KEYS : 0;
  };
  Seq q = seq(lane);
  int chunk = 1 << 30, wholes = 0, full = 0; // whole parts, units of full rounds
  bool even = true;                          // a sequence's parts as long as each other, no longer than `chunk`
  auto parts_of = [&](int tiles) { return min(max((tiles + chunk - 1) / chunk, 1), MAX_SPLITS); };
  if (p.target > 0) {
    const int room = p.target / p.Nkv, room_most = p.most / p.Nkv; // items of a K/V head
    if (ROUNDS && p.B <= 64) { // the smallest parts that all run at once, or whose rests run beside the whole ones one after another
      const int upto = scan_wave(q.blocks);
      int blocks = __builtin_amdgcn_readlane(upto, 63);
      full = blocks / room * room;
      blocks -= full;
      const int tail = min(q.blocks, max(upto - full, 0));
      const int tiles = tiles_of(q, tail), longest = max_of_wave(tiles);
      for (chunk = max(p.least, (int)(sum_of_wave((float)tail * (float)tiles) / (float)room)); longest > chunk; chunk += chunk / 16 + 1) {
        const int S = parts_of(tiles);
        wholes = sum_of_wave(tail * (S - 1));
        it.units = blocks;
        if (wholes + blocks <= room)
          break;
        if (wholes < room && chunk < longest - longest / 8) { // (less is not worth the merge)
          const int rest = tail ? tiles - (S - 1) * chunk : 0;
          even = sum_of_wave((float)tail * (float)rest) / (float)(room - wholes) + (float)max_of_wave(rest) > (float)chunk;
          if (!even)
            break;
        }
        wholes = it.units = 0;
      }
    } else {
      int tiles = tiles_of(q, q.blocks), blocks = sum_of_wave(q.blocks);
      float sum = sum_of_wave((float)q.blocks * (float)tiles); // of all units' tiles
      for (int b0 = 64; b0 < p.B; b0 += 64) {
        const Seq z = seq(b0 + lane);
        const int more = tiles_of(z, z.blocks);
        blocks += sum_of_wave(z.blocks);
        sum += sum_of_wave((float)z.blocks * (float)more);
        tiles = max(tiles, more); // (of this lane's, the longest)
      }
      const float each = sum / (float)room; // of what runs at once
      if (blocks > room && __builtin_amdgcn_ballot_w64((float)tiles > each * 1.2f) == 0) {
        // more units than that, none of them long: as they are
      } else if (p.B <= 64) { // the smallest parts that all run at once; if that leaves too much idle, more of them
        for (int items = blocks > room ? room_most : room;; items = room_most) {
          for (chunk = max(p.least, (int)(sum / (float)items)); __builtin_amdgcn_ballot_w64(tiles > chunk) != 0; chunk += chunk / 8 + 1)
            if (sum_of_wave(q.blocks * parts_of(tiles)) <= items)
              break;
          if (items == room_most || (float)chunk <= fmaxf(each * 1.4f, 2048.f / KEYS))
            break;
        }
        it.units = __builtin_amdgcn_ballot_w64(tiles > chunk) != 0 ? blocks : 0;
      } else if (room_most > blocks) { // (no more than tiles / chunk and one for each block; the sum is within 1 % of the true one)
        chunk = max(p.least, (int)(sum * 1.01f / (float)(room_most - blocks)) + 1);
        it.units = blocks;
        if constexpr (ROUNDS)
          for (int b0 = 0; b0 < p.B; b0 += 64) {
            const Seq z = b0 ? seq(b0 + lane) : q;
            wholes += sum_of_wave(z.blocks * (parts_of(tiles_of(z, z.blocks)) - 1));
          }
      }
    }
    // what these come from is the same in all lanes, which the compiler does not see (without: up to 20 % more time of the kernel)
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    wholes = __builtin_amdgcn_readfirstlane(wholes);
    even = __builtin_amdgcn_readfirstlane(even) != 0;
    it.units = __builtin_amdgcn_readfirstlane(it.units);
    it.units *= p.Nkv;
    if ((full + wholes) * p.Nkv + it.units > (int)gridDim.x || it.units < 0) // (bounds that do not ascend)
      it.units = 0;
  }
  const bool whole = ROUNDS && id >= full && id < full + wholes;
  if constexpr (ROUNDS)
    id = whole ? id - full : id < full ? id : id - wholes;
  int before = 0, other = 0; // of the counts that id is looked for in, and of the others: units, and whole parts or (not ROUNDS) all
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (b0)
      q = seq(b0 + lane);
    const int upto = ROUNDS || !p.counters ? scan_wave(q.blocks) : 0; // (with counters nobody asks for units)
    int tail = q.blocks;
    if constexpr (ROUNDS)
      tail = min(q.blocks, max(upto - full, 0)); // (full: up to 64 sequences)
    const int of_tail = tiles_of(q, tail), S = parts_of(of_tail), more = ROUNDS ? tail * (S - 1) : q.blocks * S, upto_more = scan_wave(more);
    const bool by_more = whole || !ROUNDS;
    const int sum = by_more ? upto_more : upto, sum_z = by_more ? upto : upto_more, c = by_more ? more : q.blocks, z = by_more ? q.blocks : more;
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (id < before + total) {
      const int j = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > id));
      const int blocks = __builtin_amdgcn_readlane(q.blocks, j), tiles = __builtin_amdgcn_readlane(of_tail, j);
      const int mine = before + __builtin_amdgcn_readlane(sum, j) - __builtin_amdgcn_readlane(c, j), in = id - mine;
      const int its = other + __builtin_amdgcn_readlane(sum_z, j) - __builtin_amdgcn_readlane(z, j);
      it.o.b = b0 + j;
      it.o.start = __builtin_amdgcn_readlane(q.s, j);
      it.o.n = __builtin_amdgcn_readlane(q.n, j);
      it.S = __builtin_amdgcn_readlane(S, j);
      if constexpr (ROUNDS) {
        const int split_blocks = __builtin_amdgcn_readlane(tail, j), units_before = whole ? its : mine, wholes_before = whole ? mine : its;
        const int split = whole ? in / split_blocks : 0, unit = whole ? blocks - split_blocks + in - split * split_blocks : in; // of the sequence
        if (unit < blocks - split_blocks)
          it.S = 1;
        const int part = even ? (tiles + it.S - 1) / it.S : chunk;
        it.o.at = blocks - 1 - unit;
        it.low = whole ? max(tiles - (split + 1) * part, 0) : 0;
        it.high = whole ? tiles - split * part : it.S > 1 ? tiles - (it.S - 1) * part : INT_MAX;
        it.first = (wholes_before + unit - (blocks - split_blocks)) * p.Nkv + it.hk;
        it.stride = split_blocks * p.Nkv;
        it.last = (wholes + units_before + unit - full) * p.Nkv + it.hk;
        it.mine = whole ? it.first + split * it.stride : it.last;
        it.unit = whole ? -1 : (units_before + unit - full) * p.Nkv + it.hk;
      } else {
        const int split = in / blocks;
        it.o.at = in - split * blocks;
        it.low = (int)((int64_t)(it.S - 1 - split) * tiles / it.S);
        it.high = (int)((int64_t)(it.S - split) * tiles / it.S);
        it.first = (mine + it.o.at) * p.Nkv + it.hk;
        it.stride = blocks * p.Nkv;
        it.last = it.first + (it.S - 1) * it.stride;
        it.mine = it.first + split * it.stride;
        it.unit = split < it.S - 1 ? -1 : (its + it.o.at) * p.Nkv + it.hk;
      }
      return true;
    }
    before += total;
    other += __builtin_amdgcn_readlane(sum_z, 63);
  }
  return false;
}

template <int NJ, int CG, int CW, int TW, int KEYS>
__global__ void __launch_bounds__(64 * CW * TW, CW > 1 ? 2 : 1)
paged_attn_kernel(const PagedAttnParams p) {
  constexpr int H = 32 * NJ, ROW = 64 * NJ, PER = 4 * NJ, SIDE = KEYS * ROW, WCOLS = 16 * CG, COLS = WCOLS * CW, TH = 64 * CW * TW, NA = H / 16, NT = KEYS / 16;
  constexpr int XK = NJ % 4 == 0 ? 4 : NJ % 2 == 0 ? 2 : 1, XV = NJ % 4 == 0 ? 8 : NJ % 2 == 0 ? 4 : 2, NR = NJ == 3 ? 6 : XV;
  constexpr int RUNS = 2 * NT, MINE = RUNS >= CW ? RUNS / CW : 1; // runs of 16 rows of a tile, K then V; of a wave
  static_assert((RUNS % CW == 0 || CW > RUNS) && (KEYS == 32 || KEYS == 64));
  extern __shared__ __align__(16) uint8_t lds[]; // V [team][stage], K [team][stage]
  __shared__ int arrived_last;
  __shared__ int tree[PAGED_NODES]; // parents, of a sequence that has no more (a load from memory waits for the tile under way)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % CW, team = __builtin_amdgcn_readfirstlane(tid >> 6) / CW;
  const int g = lane >> 4, c = lane & 15;
  Item it;
  const bool any = locate_item<COLS, KEYS, (TW == 1 && CW > 1)>(p, (int)blockIdx.x, it);
  if (p.target > 0 && !p.counters && tid == 0 && blockIdx.x == 0)
    merges_of<COLS, H>(p)->S = it.units;
  if (!any)
    return;
  const Block& o = it.o;
  const int hk = it.hk, col0 = o.at * COLS, ncol = min(COLS, o.n * p.R - col0); // of this workgroup
  const int past = paged_past(p, o.b), keys = paged_keys(p, past, (col0 + ncol - 1) / p.R); // that some column sees
  const int tiles = (keys + KEYS - 1) / KEYS, S = it.S;
  const bool idle = wave * WCOLS >= ncol;
  if (tid == 0 && !p.counters && it.unit >= 0 && it.unit < it.units)
    merges_of<COLS, H>(p)[1 + it.unit] = Merge{S, it.first, it.stride, it.last, hk, o.start, col0, ncol};
  const int32_t* const parents = p.parents ? p.parents + o.start : nullptr;
  int node[CG], up[CG]; // of this lane's columns; where their ways up have come to
  bf16x8 q[CG][NJ];
#pragma unroll
  for (int k = 0; k < CG; k++) {
    const int col = col0 + min(wave * WCOLS + k * 16 + c, ncol - 1);
    node[k] = up[k] = col / p.R;
    const uint16_t* qrow = p.q + (int64_t)(o.start + node[k]) * p.q_ld + (hk * p.R + col - node[k] * p.R) * H + g * 8;
#pragma unroll
    for (int j = 0; j < NJ; j++)
      q[k][j] = *reinterpret_cast<const bf16x8*>(qrow + j * 32);
  }
  // Tiles top, top - TW, .. of this team, down to the part's last one.
  const int low = it.low, top = min(it.high, tiles) - 1 - team, most = (top + team - low) / TW + 1;
  const ConstantInts table = (ConstantInts)(uintptr_t)(p.g.table + (int64_t)o.b * p.g.table_ld);
  const int64_t values = (((int64_t)p.g.pages * p.Nkv) << p.g.shift) * H;
  int ids[MINE]; // pages of this wave's runs of the tile that is asked for next
  auto look_up = [&](int t) {
    if (t >= low) {
#pragma unroll
      for (int i = 0; i < MINE; i++) {
        const int run = (i * CW + wave) % NT; // (more waves than runs: the last ones bring nothing)
        ids[i] = table[min(t * KEYS + run * 16, keys - 1) >> p.g.shift];
      }
    }
  };
  uint32_t from[2][NJ]; // offset of this lane's chunk in a run's rows: K, V
#pragma unroll
  for (int s = 0; s < 2; s++)
#pragma unroll
    for (int i = 0; i < NJ; i++) {
      const int item = i * 64 + lane, row = item / PER, ch = item % PER;
      from[s][i] = (uint32_t)(row * ROW + (ch ^ (s ? packed_v_turn(NJ, row) : packed_k_turn(NJ, row))) * 16);
    }
  auto request = [&](int t, int stage) __attribute__((always_inline)) {
    const bool whole = (t + 1) * KEYS <= keys; // (rows past the keys repeat the last one)
    auto runs = [&](auto whole_) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole_)::value;
      static_for<0, MINE>([&](auto I) {
        constexpr int i = decltype(I)::value;
        const int run = (i * CW + wave) % NT, side = (i * CW + wave) / NT;
        if (CW > RUNS && side > 1)
          return;
        const int key = WHOLE ? t * KEYS + run * 16 : min(t * KEYS + run * 16, keys - 1), rows = WHOLE ? 16 : min(keys - key, 16);
        // (a page that does not exist: the first one)
        const int id = (unsigned)ids[i] < (unsigned)p.g.pages ? ids[i] : 0;
        const uint16_t* const at = p.layer + (side ? values : 0) + slot_at(p.g, id, p.Nkv, hk, key, H);
        const auto src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), 0, rows * ROW, 0x00020000);
        uint8_t* const dst = lds + (((side ? 0 : TW) + team) * 2 + stage) * SIDE + run * (NJ * 1024);
        static_for<0, NJ>([&](auto J) {
          constexpr int j = decltype(J)::value;
          const uint32_t k_off = from[0][j], v_off = from[1][j];
          uint32_t off = side ? v_off : k_off;
          if constexpr (!WHOLE)
            off -= (uint32_t)(max((j * 64 + lane) / PER - (rows - 1), 0) * ROW);
          load_to_lds(src, dst + j * 1024, off);
        });
      });
    };
    if (whole)
      runs(std::true_type{});
    else
      runs(std::false_type{});
  };
  uint32_t kaddr[XK], vaddr[XV];
#pragma unroll
  for (int j = 0; j < XK; j++)
    kaddr[j] = (uint32_t)((TW + team) * 2 * SIDE + c * ROW + ((j * 4 + g) ^ packed_k_turn(NJ, c)) * 16);
  {
    const int r = g * 4 + (c >> 2);
#pragma unroll
    for (int d = 0; d < XV; d++)
      vaddr[d] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds +
                 (uint32_t)(team * 2 * SIDE + r * ROW + ((d * 2 + ((c >> 1) & 1)) ^ packed_v_turn(NJ, r)) * 16 + (c & 1) * 8);
  }

  float m[CG], l[CG];
  f32x4 acc[CG][NA];
#pragma unroll
  for (int k = 0; k < CG; k++) {
    m[k] = LOWEST;
    l[k] = 0.f;
#pragma unroll
    for (int dt = 0; dt < NA; dt++)
      acc[k][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float unit = p.scale * LOG2E;
  const bool small = o.n <= PAGED_NODES;
  if (parents && small)
    for (int i = tid; i < o.n; i += TH)
      tree[i] = parent_of(parents, i);
  auto parent = [&](int i) { return small ? tree[i] : parent_of(parents, i); };
  auto tile = [&](auto S_, int t, int highest) __attribute__((always_inline)) { // highest: the tile of the first team, at the same time
    constexpr int stage = decltype(S_)::value;
    const int kb = t * KEYS;
    // this tile has landed and the other stage has been read, for this wave and then for every wave that shares them (the wait as a
    // builtin, which the compiler counts: behind one in asm it waits for q once more in every tile, and so for the loads under way)
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0)
    if constexpr (CW > 1)
      __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    const bool mine = t >= low; // (uniform in a team)
    bool odd = false;
    if ((CW == 1 ? kb : highest * KEYS) + KEYS > past) { // some column may not see some key
      if (mine) {
#pragma unroll
        for (int i = 0; i < (KEYS * PER + 64 * CW - 1) / (64 * CW); i++) {
          const int at = i * 64 * CW + wave * 64 + lane;
          if (KEYS * PER % (64 * CW) != 0 && at >= KEYS * PER)
            continue;
          const i32x4 w = *(reinterpret_cast<const i32x4*>(lds + (team * 2 + stage) * SIDE) + at);
#pragma unroll
          for (int j = 0; j < 4; j++)
            odd |= mx4_non_finite((uint32_t)w[j]);
        }
      }
      odd = CW == 1 ? __builtin_amdgcn_ballot_w64(odd) != 0 : __syncthreads_or(odd);
    }
    if (t - TW >= low) {
      request(t - TW, stage ^ 1); // in flight during the arithmetic below
      look_up(t - 2 * TW);
    }
    f32x4 sc[CG][NT];
    uint64_t seen[CG];
#pragma unroll
    for (int k = 0; k < CG; k++)
      seen[k] = ~0ull; // (a tile below the step's slots beside one that holds some)
    const bool busy = mine && !idle;
    if (busy) {
      const uint8_t* const st = lds + stage * SIDE;
#pragma unroll
      for (int u = 0; u < NT; u++) {
#pragma unroll
        for (int k = 0; k < CG; k++)
          sc[k][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          const bf16x8 w = *reinterpret_cast<const bf16x8*>(st + kaddr[j % XK] + u * (16 * ROW) + j / XK * (XK * 64));
#pragma unroll
          for (int k = 0; k < CG; k++)
            sc[k][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, q[k][j], sc[k][u], 0, 0, 0);
        }
      }
      if (kb + KEYS > past) { // (uniform in a team)
        const int lo = kb - past; // the node whose slot is the tile's first key
#pragma unroll
        for (int k = 0; k < CG; k++) {
          uint64_t s = lo < 0 ? (1ull << -lo) - 1 : 0ull; // (above -KEYS)
          if (!parents) {
            const int last = node[k] - lo; // (the capacity ends the keys: what lies behind is not asked about)
            s = last >= 63 ? ~0ull : last < 0 ? 0ull : (2ull << last) - 1;
          } else {
            while (up[k] >= max(lo + KEYS, 0))
              up[k] = parent(up[k]);
            while (up[k] >= max(lo, 0)) {
              s |= 1ull << (up[k] - lo);
              up[k] = parent(up[k]);
            }
          }
          const int behind = keys - kb;
          if (behind < 64)
            s &= (1ull << behind) - 1;
          seen[k] = s;
          const uint64_t bits = s >> (g * 4);
#pragma unroll
          for (int i = 0; i < 4 * NT; i++)
            sc[k][i >> 2][i & 3] = bits >> ((i >> 2) * 16 + (i & 3)) & 1 ? sc[k][i >> 2][i & 3] : -INFINITY;
        }
      }
#pragma unroll
      for (int k = 0; k < CG; k++) {
        float mx = m[k];
#pragma unroll
        for (int i = 0; i < 4 * NT; i++)
          mx = fmaxf(mx, sc[k][i >> 2][i & 3]);
        // Few columns: the maximum is followed at once; many: once it is 2^8 above (relative error against 64 bits 1.8e-3 and 2.2e-3)
        if (__builtin_amdgcn_ballot_w64((mx - m[k]) * unit > (COLS <= 32 ? 0.f : 8.f)) != 0) {
          mx = max_of_groups(mx);
          const float alpha = __builtin_amdgcn_exp2f((m[k] - mx) * unit);
#pragma unroll
          for (int dt = 0; dt < NA; dt++)
            acc[k][dt] *= alpha;
          l[k] *= alpha;
          m[k] = mx;
        }
      }
    }
    if (__builtin_expect(odd, 0)) { // values that are not finite: to the columns that see them, then zeros
      uint8_t* const vt = lds + (team * 2 + stage) * SIDE;
      if (busy) {
#pragma unroll 1
        for (int key = 0; key < KEYS; key++)
#pragma unroll
          for (int dt = 0; dt < NA; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int ch = dt * 16 + g * 4 + e;
              const uint32_t w = *reinterpret_cast<const uint16_t*>(vt + key * ROW + ((ch >> 3) ^ packed_v_turn(NJ, key)) * 16 + (ch & 7) * 2);
#pragma unroll
              for (int k = 0; k < CG; k++)
                if ((w & 0x7f80u) == 0x7f80u && (seen[k] >> key & 1))
                  acc[k][dt][e] += bf16_bits_to_f32(w);
            }
      }
      if constexpr (CW > 1)
        __syncthreads();
      if (mine) {
        for (int at = wave * 64 + lane; at < KEYS * PER; at += 64 * CW) {
          i32x4* const it = reinterpret_cast<i32x4*>(vt) + at;
          const i32x4 w = *it;
          *it = i32x4{(int)mx4_finite((uint32_t)w[0]), (int)mx4_finite((uint32_t)w[1]), (int)mx4_finite((uint32_t)w[2]), (int)mx4_finite((uint32_t)w[3])};
        }
      }
      if constexpr (CW > 1)
        __syncthreads();
      else
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    }
    if (busy) {
      bf16x8 pb[CG][NT / 2];
      auto weights = [&](int u) __attribute__((always_inline)) { // of 32 keys
#pragma unroll
        for (int k = 0; k < CG; k++) {
          const float off = -m[k] * unit;
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const f32x4 v = sc[k][u * 2 + (i >> 2)];
            const bf16x2 pr = {(__bf16)__builtin_amdgcn_exp2f(fmaf(v[i & 3], unit, off)), (__bf16)__builtin_amdgcn_exp2f(fmaf(v[(i & 3) + 1], unit, off))};
            l[k] = __builtin_amdgcn_fdot2_f32_bf16(pr, bf16x2{(__bf16)1.f, (__bf16)1.f}, l[k], false);
            pb[k][u][i] = pr[0];
            pb[k][u][i + 1] = pr[1];
          }
        }
      };
      weights(0);
      static_for<0, KEYS / 32>([&](auto U) {
        constexpr int u = decltype(U)::value;
        static_for<0, NA / NR>([&](auto D) { // NR pieces of channels
          constexpr int d0 = decltype(D)::value * NR;
          i32x2 vv[NR][2];
          packed_v_operands<stage * SIDE + u * 32 * ROW + d0 * 32, 16 * ROW>(vv, vaddr);
          if constexpr (d0 == 0 && u + 1 < KEYS / 32)
            weights(u + 1); // (the compiler lets them run beside the MFMAs)
#pragma unroll
          for (int d = 0; d < NR; d++) {
            const i32x4 w = {vv[d][0][0], vv[d][0][1], vv[d][1][0], vv[d][1][1]};
#pragma unroll
            for (int k = 0; k < CG; k++)
              acc[k][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), pb[k][u], acc[k][d0 + d], 0, 0, 0);
          }
        });
      });
    }
  };
  if (top >= low) {
    look_up(top);
    request(top, 0);
    look_up(top - TW);
  }
  if (parents)
    __syncthreads();
  for (int k = 0; k < most; k += 2) {
    tile(std::integral_constant<int, 0>{}, top - k * TW, top + team - k * TW);
    if (k + 1 < most)
      tile(std::integral_constant<int, 1>{}, top - (k + 1) * TW, top + team - (k + 1) * TW);
  }
#pragma unroll
  for (int k = 0; k < CG; k++) {
    l[k] += __shfl_xor(l[k], 16);
    l[k] += __shfl_xor(l[k], 32);
    m[k] = m[k] == LOWEST ? LOWEST : m[k] * unit; // in powers of two
  }

  auto store4 = [&](int cc, int ch, f32x4 v, float sum) { // (nothing seen: zeros)
    const int cl = col0 + cc, nd = cl / p.R, rr = cl - nd * p.R;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    *reinterpret_cast<uint2*>(p.out + ((int64_t)(o.start + nd) * p.Nq + hk * p.R + rr) * H + ch) =
        make_uint2(f32x2_to_bf16_bits(v[0] * inv, v[1] * inv), f32x2_to_bf16_bits(v[2] * inv, v[3] * inv));
  };
  // A split's results for the merge: stores and loads at the scope of the device, written through to the level that all XCDs share.
  constexpr int SHARED = 16; // (sc1)
  const auto part = __builtin_amdgcn_make_buffer_rsrc(p.part, 0, p.parts * (COLS * H * 4), 0x00020000);
  const auto part_ml = __builtin_amdgcn_make_buffer_rsrc(p.part + (int64_t)p.parts * COLS * H, 0, p.parts * (COLS * 8), 0x00020000);
  if (TW == 1 && S == 1) {
#pragma unroll
    for (int k = 0; k < CG; k++) {
      const int cc = wave * WCOLS + k * 16 + c;
      if (cc < ncol)
#pragma unroll
        for (int dt = 0; dt < NA; dt++)
          store4(cc, dt * 16 + g * 4, acc[k][dt], l[k]);
    }
  } else { // the teams' states through LDS
    constexpr int OP = H + 4;
    float* const mo = reinterpret_cast<float*>(lds); // [team][col][OP]
    float* const sm = mo + TW * COLS * OP;           // [team][col] maximum, then sum
    __syncthreads();
#pragma unroll
    for (int k = 0; k < CG; k++) {
      const int cc = wave * WCOLS + k * 16 + c;
#pragma unroll
      for (int dt = 0; dt < NA; dt++)
        if (cc < ncol)
          *reinterpret_cast<f32x4*>(mo + (team * COLS + cc) * OP + dt * 16 + g * 4) = acc[k][dt];
      if (g == 0) {
        sm[team * COLS + cc] = m[k];
        sm[TW * COLS + team * COLS + cc] = l[k];
      }
    }
    __syncthreads();
    for (int i = tid; i < ncol * (H / 4); i += TH) {
      const int cl = i / (H / 4), d4 = i % (H / 4);
      float M = sm[cl];
#pragma unroll
      for (int w = 1; w < TW; w++)
        M = fmaxf(M, sm[w * COLS + cl]);
      float Ls = 0.f;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < TW; w++) {
        const float wt = __builtin_amdgcn_exp2f(sm[w * COLS + cl] - M);
        Ls = fmaf(wt, sm[TW * COLS + w * COLS + cl], Ls);
        const f32x4 ow = *reinterpret_cast<const f32x4*>(mo + (w * COLS + cl) * OP + d4 * 4);
#pragma unroll
        for (int e = 0; e < 4; e++)
          v[e] = fmaf(wt, ow[e], v[e]);
      }
      if (S == 1) {
        store4(cl, d4 * 4, v, Ls);
      } else {
        const int at = it.mine * COLS + cl;
        if (p.counters) {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part, (at * H + d4 * 4) * 4, 0, SHARED);
          if (d4 == 0)
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(M, Ls)), part_ml, at * 8, 0, SHARED);
        } else {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part, (at * H + d4 * 4) * 4, 0, 0);
          if (d4 == 0)
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(M, Ls)), part_ml, at * 8, 0, 0);
        }
      }
    }
  }
  if (S == 1 || !p.counters)
    return;
  // The split that arrives last merges all of them, in split order (the same sums whichever that is).  Every thread waits until
  // its own stores are acknowledged, then the barrier, the arrival, and the device-scope loads; nobody waits for another workgroup.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    arrived_last = atomicInc(p.counters + (int64_t)it.last * MX4_COUNTER_STRIDE, (unsigned)S - 1) == (unsigned)S - 1;
  __syncthreads();
  if (!arrived_last)
    return;
  // A load at that scope takes more than a microsecond: those of the first eight parts are under way while the weights are found.
  const int lane_ = tid & 63, wave_ = tid >> 6;
  f32x4 a[8];
  auto fetch = [&](int i, int s0) {
    const int cc = i / (H / 4), d4 = i % (H / 4);
#pragma unroll
    for (int u = 0; u < 8; u++) // (past the last one: that again)
      a[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, (it.part(min(s0 + u, S - 1)) * COLS + cc) * (H * 4) + d4 * 16, 0, SHARED));
  };
  if (tid < ncol * (H / 4))
    fetch(tid, 0);
  float* const merged = reinterpret_cast<float*>(lds); // [col][MAX_SPLITS + 1]: weights of the splits, then the sum
  for (int cc = wave_; cc < ncol; cc += TH / 64) { // a lane per split
    float2 ml = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(part_ml, (it.part(min(lane_, S - 1)) * COLS + cc) * 8, 0, SHARED));
    if (lane_ >= S)
      ml = float2{LOWEST, 0.f};
    float M = ml.x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
      M = fmaxf(M, __shfl_xor(M, d));
    const float wt = __builtin_amdgcn_exp2f(ml.x - M), Ls = wave_sum(wt * ml.y);
    merged[cc * (MAX_SPLITS + 1) + lane_] = wt;
    if (lane_ == 0)
      merged[cc * (MAX_SPLITS + 1) + MAX_SPLITS] = Ls;
  }
  __syncthreads();
  for (int i = tid; i < ncol * (H / 4); i += TH) {
    const int cc = i / (H / 4), d4 = i % (H / 4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += 8) {
      if (i != tid || s0)
        fetch(i, s0);
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (s0 + u < S) {
          const float wt = merged[cc * (MAX_SPLITS + 1) + s0 + u];
#pragma unroll
          for (int e = 0; e < 4; e++)
            v[e] = fmaf(wt, a[u][e], v[e]);
        }
    }
    store4(cc, d4 * 4, v, merged[cc * (MAX_SPLITS + 1) + MAX_SPLITS]);
  }
}

// The parts' results, where the launch itself does not merge them: a thread takes four channels of a column, all parts.  Bound by their bytes,
// 8 H fp32 a column and part there and back, and a launch: 4 us for 28 units of nine parts, 7.5 for 248 of two or three (128 columns each).
template <int NJ, int COLS>
__global__ void __launch_bounds__(256)
paged_merge_kernel(const PagedAttnParams p) {
  constexpr int H = 32 * NJ, EACH = H / 4, PER = 256 / EACH; // threads of a column, columns of a workgroup
  const Merge* const all = merges_of<COLS, H>(p);
  const int units = all->S;
  const Merge it = all[1 + blockIdx.x];
  if ((int)blockIdx.x >= units || it.S == 1)
    return;
  const int S = it.S;
  const int d4 = (int)threadIdx.x % EACH;
  if ((int)threadIdx.x >= PER * EACH)
    return;
  for (int cc = (int)blockIdx.y * PER + (int)threadIdx.x / EACH; cc < it.ncol; cc += (int)gridDim.y * PER) {
    const float* const part = p.part + cc * H + d4 * 4;
    const float2* const ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.parts * COLS * H) + cc;
    float M = LOWEST, L = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += 8) { // eight parts' loads at a time
      float2 z[8];
      f32x4 a[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int64_t i = (int64_t)(s0 + u < S - 1 ? it.first + (s0 + u) * it.stride : it.last) * COLS;
        z[u] = ml[i];
        a[u] = *reinterpret_cast<const f32x4*>(part + i * H);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < 8; u++)
        top = fmaxf(top, z[u].x);
      const float alpha = __builtin_amdgcn_exp2f(M - top);
      M = top;
      L *= alpha;
      v *= alpha;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const float w = s0 + u < S ? __builtin_amdgcn_exp2f(z[u].x - M) : 0.f;
        L = fmaf(w, z[u].y, L);
#pragma unroll
        for (int e = 0; e < 4; e++)
          v[e] = s0 + u < S ? fmaf(w, a[u][e], v[e]) : v[e];
      }
    }
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    const int cl = it.col0 + cc, nd = cl / p.R;
    *reinterpret_cast<uint2*>(p.out + ((int64_t)(it.start + nd) * p.Nq + it.hk * p.R + cl - nd * p.R) * H + d4 * 4) =
        make_uint2(f32x2_to_bf16_bits(v[0] * inv, v[1] * inv), f32x2_to_bf16_bits(v[2] * inv, v[3] * inv));
  }
}

// ---------------------------------------------------------------------------
// The keys and values of an accepted path to the slots from past on, in all layers.  A thread takes 16 bytes of a head's row through the
// whole path: node path[i] goes to slot past + i, and as path ascends no row is read after another was written over it.  Launch and one way
// through table, path and rows: one sequence, 4 layers 2.1 us; 12 sequences, 28 layers (5.5 MB) 4.2.
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
  const int first = p.cu ? p.cu[b] : b, n = p.cu ? min(max(p.cu[b + 1], 0), p.T) - max(first, 0) : 1;
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

static int attn_launch(const char* who, PagedAttnParams& p, int H, int64_t ws_bytes, int64_t counter_bytes, hipStream_t stream) {
  hipError_t e = hipSuccess;
  int rc = TPPX_OK;
  auto at_once = [](size_t lds) { return (int64_t)256 * std::min<int64_t>(160 * 1024 / lds, 8); }; // workgroups of one wave a team
  auto go = [&](auto nj, auto cg, auto cw, auto tw, auto kt) {
    constexpr int NJ = decltype(nj)::value, CG = decltype(cg)::value, CW = decltype(cw)::value, TW = decltype(tw)::value, KEYS = decltype(kt)::value, COLS = 16 * CG * CW;
    const int64_t blocks = p.cu ? ((int64_t)p.T * p.R + (int64_t)p.B * (COLS - 1)) / COLS : (int64_t)p.B * ((p.R + COLS - 1) / COLS);
    const int64_t units = blocks * p.Nkv;
    if (units > ((int64_t)1 << 31) / (64 * CW * TW)) { // (threads of a grid)
      rc = set_error(TPPX_ESHAPE, "%s: problem too large", who);
      return;
    }
    const size_t stages = 4 * TW * KEYS * 64 * (size_t)NJ;
    const int64_t room = std::min<int64_t>(std::max<int64_t>(ws_bytes - (int64_t)sizeof(Merge), 0) / (COLS * (32 * NJ + 2) * (int64_t)sizeof(float) + (int64_t)sizeof(Merge)), (((int64_t)1 << 31) - 1) / (COLS * 32 * NJ * 4));
    // What runs at once, by the LDS.  Twice that, and the merge has more to do than it gives: one token behind 30000 keys 36.4 us, so 30.5; 8
    // behind up to 8000 22.1 and 17.3.
    int64_t target = env_int("TPPX_PAGED_ITEMS", 0);
    if (target <= 0)
      target = CW > 1 ? 256 * (TW == 1 || stages <= 80 * 1024 ? 2 : 1) : at_once(stages);
    // no more than the capacity would make: a workgroup without work waits for room on a CU like any other
    const int64_t capacity = p.g.table_ld << p.g.shift, limit = std::min<int64_t>(room, ((int64_t)1 << 31) / (64 * CW * TW));
    // Parts of 512 keys at least where the launch merges them (one token behind 400 keys 8.6 us, of 256 10.0; behind 1900 12.3 and 12.0), of
    // 256 else (8 nodes behind 1000 keys 11.4 us, of 512 13.2).
    p.least = std::max(env_int("TPPX_PAGED_LEAST", COLS == 16 && !p.cu ? 512 : 256) / KEYS, 1);
    target = std::min<int64_t>({target, limit, units * ((capacity / KEYS + p.least) / p.least)});
    const bool rounds = TW == 1 && CW > 1 && p.B <= 64;
    int64_t most; // (rounds: whole parts are fewer than `target`, and so are the units that are split)
    if (rounds) {
      target = std::min(target, room / 2);
      most = 2 * target;
    } else { // (few units: parts of equal lengths come near enough to the same)
      most = std::min<int64_t>({4 * units <= target || capacity < 4096 ? std::max(target, units + p.Nkv) : (units / target + 2) * target, limit, units * ((capacity / KEYS + p.least) / p.least)});
    }
    // A few pages hold no more than a part would: not worth the look at the lengths and the merge (8 nodes behind 300 keys 8.7 us; 440 keys
    // in parts of 256 11.3, whole 9.8).
    if (target < p.Nkv || (!rounds && most < units + p.Nkv) || capacity <= 384)
      target = most = 0;
    p.target = (int)target;
    p.most = p.parts = (int)most;
    const int64_t items = rounds ? target + units : std::max<int64_t>(most, units);
    // Merged in the launch, by the part that arrives last (counters), where a unit is a few rows: single tokens (1 behind 1900 keys 12.3 us, by a
    // second launch 13.3; 8 behind up to 8000 17.2 and 18.3)
    const bool here = COLS == 16 && p.R <= 16 && !p.cu && p.parts * MX4_COUNTER_STRIDE * (int64_t)sizeof(unsigned) <= counter_bytes;
    if (!here)
      p.counters = nullptr;
    const size_t teams = TW > 1 || target ? TW * COLS * (32 * NJ + 6) * sizeof(float) : 0; // (the merge's weights take less)
    const size_t lds = std::max(stages, teams);
    auto kern = paged_attn_kernel<NJ, CG, CW, TW, KEYS>;
    e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds);
    if (e != hipSuccess)
      return;
    kern<<<dim3((unsigned)items), dim3(64 * CW * TW), lds, stream>>>(p);
    constexpr int PER = 256 / (8 * NJ);
    if (target && !here) { // (units that were not split end at once: not too many of those)
      const int64_t split = rounds ? std::min(target, units) : units;
      paged_merge_kernel<NJ, COLS><<<dim3((unsigned)split, (unsigned)std::min<int64_t>((COLS + PER - 1) / PER, std::max<int64_t>(4096 / split, 1))), dim3(256), 0, stream>>>(p);
    }
  };
  const int64_t cols = (p.cu ? (p.T + p.B - 1) / p.B : 1) * (int64_t)p.R; // of a sequence's K/V head, on average
  // units of c columns, about: pieces of prompts as if they were equally long, the last block of a tree half empty
  auto units_of = [&](int64_t c) { return (p.parents ? ((int64_t)p.T * p.R + (int64_t)p.B * (c / 2)) / c : (cols + c - 1) / c * (int64_t)p.B) * p.Nkv; };
  constexpr std::integral_constant<int, 1> n1{};
  constexpr std::integral_constant<int, 2> n2{};
  constexpr std::integral_constant<int, 4> n4{};
  constexpr std::integral_constant<int, 32> k32{};
  constexpr std::integral_constant<int, 64> k64{};
  // Forms (columns of a workgroup; teams).  2 (32; 4): 12 x 4 nodes behind 3000 keys of 64 heads on 8 22.0 us (1: 23.8, 4: 26.8).  3 (64; 4): few
  // units, as teams share their tiles: 64 behind 8000 36.6 (4: 39.5), 4 x 128 behind 1000 of 32 on 32 26 (4: 30).  4 (128; 1): an operand
  // read feeds 32 columns and nothing is merged in LDS: 128 behind 8000 53.5 (3: 60), 1024 282 (3: 392).  Heads of 192 and 256 have
  // registers for 16 columns a wave: no form 2 (2 x 20 behind 1500 of 16 on 16: 3 17.8, 1 22.5).
  // 16 columns: single tokens, and little work altogether.  1 (four teams, two at heads of 192 and 256): 8 nodes behind 50, 2000, 8000 keys 7.1, 11.4,
  // 18.4 (3: 10.5, 15.2, 21.8); 60 behind 5000 of 28 on 4 over 25.8 (3: 22.3).  5 (two), 6 (one): more units than workgroups with more
  // teams run at once, and short ones: 24 x 3 behind 300 5 10.9 (1: 13.3, 3: 11.4), 18 single tokens without a past of 32 on 32 6 5.8 (5: 9.6, 1: 14),
  // 3 x 69 without a past 6 9.4 (1: 16, 3: 10.1), 64 single tokens behind 500 5 15.5 (1: 17.9, 6: 18.8), behind 2000 1 49.8 (5: 53.6).
  const int form = env_int("TPPX_PAGED_FORM", 0);
  mx4_for_head(H, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    const int64_t capacity = p.g.table_ld << p.g.shift;
    const int64_t u16 = units_of(16);
    auto room = [&](int teams) { return at_once(teams * 8192 * NJ); };
    int f = form;
    if (!f && cols <= 16) {
      f = 1;
      if (u16 > room(NJ > 4 ? 2 : 4) && capacity <= 1024) { // rounds of: start and end, tiles (us, as measured)
        auto cost = [&](int teams) { return (double)((u16 + room(teams) - 1) / room(teams)) * ((teams > 1 ? 5.5 : 4.5) + 0.0034 * NJ * (double)capacity / teams); };
        const double one = cost(1), two = cost(2), four = NJ > 4 ? two : cost(4);
        f = one < two && one < four ? 6 : two < four ? 5 : 1;
      }
    } else if (!f && NJ <= 4) {
      if (u16 <= room(4) && u16 * capacity * NJ < 1600000)
        f = 1;
      else if (u16 <= room(2) && capacity > 128 && capacity <= 512)
        f = 5;
      else if (u16 <= room(1) && capacity <= 128)
        f = 6;
      else if (cols <= 32)
        f = 2;
    }
    if (!f)
      f = units_of(64) <= 280 && units_of(64) * capacity < 800000 ? 3 : 4;
    if constexpr (NJ > 4) {
      if (f == 6)
        go(nj, n1, n1, n1, k32);
      else if (f == 1 || f == 5)
        go(nj, n1, n1, n2, k32);
      else if (f == 4)
        go(nj, n1, n4, n1, k32);
      else
        go(nj, n1, n4, n2, k32);
    } else {
      if (f == 1)
        go(nj, n1, n1, n4, k32);
      else if (f == 5)
        go(nj, n1, n1, n2, k32);
      else if (f == 6)
        go(nj, n1, n1, n1, k32);
      else if (f == 2)
        go(nj, n2, n1, n4, k32);
      else if (f == 3)
        go(nj, n2, n2, n4, k32);
      else
        go(nj, n2, n4, n1, k64);
    }
  });
  if (rc)
    return rc;
  return check_hip(e != hipSuccess ? e : hipGetLastError(), who);
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
  // heads over up to 1024 workgroups (24 trees 10.2 us; 256 13.3, 4096 12.3)
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
  p.T = (int)T; p.B = (int)B; p.Nq = (int)Nq; p.Nkv = (int)Nkv; p.R = (int)(Nq / Nkv);
  p.scale = 1.0f / sqrtf((float)H);
  p.part = (float*)ws;
  p.counters = (unsigned int*)counters;
  return attn_launch(who, p, (int)H, ws_bytes, counter_bytes, (hipStream_t)stream);
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
