// Attention of new tokens over a paged K/V cache on gfx950 MFMA: chunks of a
// prompt, single tokens, or both in one packed batch.
//
// No reference counterpart: its decode reads a contiguous cache and one query
// row per sequence (csrc/decode.cu:50-138 of shrvan30/flash-attention-cuda).
//
// Mathematics. Token t of sequence b (n_b new tokens, length L_b with them)
// sits at position p = L_b - n_b + t and sees keys 0..p:
//   o = sum_j P_j v_j / sum_j P_j,  P_j = 2^(c s_j - m),  s_j = q . k_j,
// c = scale log2 e, m a running bound of the row's c s_j (online softmax).
//
// Decomposition
//   item   = (sequence, K/V head, tile of its query rows). A row is one (token,
//            query head) pair of the K/V head's group, so an item reads K and V
//            once for the whole group. A sequence of at most 32 rows is one "narrow"
//            item; others are tiles of up to 128 rows of whole tokens.
//   share  = the items laid end to end, weighted by the keys they see, are cut
//            into equal shares, one per block (two or three blocks per CU):
//            ragged lengths and few sequences fill the chip alike, without a
//            host that knows the lengths. Each wave finds its block's share
//            from seq_lens and cu_tokens (1 us: kernel arguments, lengths, a
//            sum over the lanes, 32-bit arithmetic).
//   merge  = an item that a share's border cuts leaves one fp32 partial (O, m,
//            l) per share in the workspace. They are joined along a fixed tree (wide: in
//            pairs, narrow: 16 at a time) by whichever block is there last, so results
//            do not depend on timing (a second launch for it took 2.6 to 18.7 us).
//
// Block: 256 threads, 4 waves.
//   wide item: wave w owns query rows [32 w, +32); the waves share 64-key K and V
//     tiles in an LDS ring filled by direct global->LDS loads.
//   narrow item: the waves take key tiles in turn, each with K and V tiles of its
//     own in LDS (no barrier in the loop), and join their states at the end.
//   Products on v_mfma_f32_32x32x16 (wide; mfma_tile.h) and 16x16x32 (narrow): S^T = K Q^T,
//   O^T += V^T P^T, so a query row's scores lie in one lane pair, or four lanes.
//
// Roundings to 16 bits. P is rounded once on wide items (the row sum is taken of
// the rounded weights, so a row that one key carries is exact) and split into two
// parts on narrow ones, where memory is what bounds the loop: against 64 bits (relative
// 2-norm, N(0,1)) fp16 outputs of wide items are 2.6e-4 to 2.9e-4 off, of narrow ones
// 2.0e-4 (the output's own rounding); bf16 2.3e-3 and 1.7e-3. Split on wide items too, P
// costs the prompt below 74 us for 56.5 and the long chunks 686 for 508 (one box).
//
// Measured (us per call among others; B sequences, H / H_kv heads, D head_dim):
//   B1 H12 D64, 512 keys, one token             7.3   chain of a block's loads
//   B32 H14/2 D64, 4096 keys ragged, one token 14.0   2.5 TB/s: share 2 us, ~4 rounds of
//                                                     loads, publish and join 2 us
//   B8 H32/8 D128 bf16, 8191 ragged, one token 31.1   4.9 TB/s of K and V: HBM
//   B1 H14 D64, prompt of 4096                 53.1   566 TFLOP/s; MFMA 23 %, VALU 35 % busy: a
//                                                     wave does one after the other
//   B24 H28/4 D128, 3 chunks to 777 + tokens   47.5   2.7 TB/s and 340 TFLOP/s; its chunks alone 42
//   B4 H32/8 D128 bf16, chunks to 2048 on 6144  484   932 TFLOP/s; MFMA 49 %, VALU 36 % busy:
//                                                     the two hardly run at once
//
// Memory safety. Lengths, bounds and page ids are device data, which the host
// cannot check: token ranges are clamped to the packed tensors, key ranges to the
// page table's width, and a page id outside the pool is replaced by page 0 for
// the address and its keys are masked out. V rows past a sequence's end
// are cleared in LDS before they meet a weight of zero (0 * NaN); what a query may not
// see for its position does not reach it either (wide_pass).

#include "mfma_tile.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kTileKeys = 64;     // keys per tile of a wide item, and the unit of a share's border
constexpr int kWideRows = 128;    // query rows of a wide item
constexpr int kNarrowRows = 32;   // most query rows of a narrow item
constexpr int kNarrowKeys = 32;   // keys of a narrow item's tile, of which each wave has its own

// Weights of the shares, measured over the cases above and 16 random batches:
// An item's fixed cost (start, partial, join) in keys: 320 where there are many (192: B8
// H32/8 D128 33.5 us for 32.0, mixed 54.0 for 52.5; 128: mixed 61; 384 as 320), and
// 512, the least share, where there are blocks to spare, so that no block takes two items
// (13 prompts of ~138 tokens 21.4 -> 12.9 us, 24 short sequences 11.4 -> 7.7).
constexpr int kItemKeys = 320;
constexpr int kFewItemKeys = 512;
// Least weight of a share: 512 keys (256: two sequences of 8k keys 19.0 us for 16.9;
// 640 and more: 32 ragged sequences 15.9 for 15.0).
constexpr int kMinShareKeys = 512;
// Borders inside wide items lie at multiples of this many tiles (1 alike; 4: prompt 62 us
// for 57), inside narrow ones at a round of the block's waves; items of at most kWholeSteps
// such steps are never cut, since a cut costs about as much as two of them.
constexpr int kWideStep = 2;
constexpr int kWholeSteps = 4;
// Narrow items of more pieces are joined in groups of 16 first (one sequence of 131072 keys of
// 14/2 heads 42.2 -> 21.7 us, of 524288 82.4 -> 53.4; with 16 here two sequences of 17
// pieces each 19.7 us for 16.3).
constexpr int kFlatPieces = 48;

// Blocks per CU and LDS for tiles per block, by head size. A head_dim 64 wave fits 168
// VGPRs, so three blocks share a CU (two: prompt 57.3 us for 55.4, 20 sequences with 4
// chunks 48.2 for 45.4). At head_dim 128, one block of 8 waves with 256-row items instead of
// two of 4 halves the tile loads (long chunks 477 us for 496, long tokens 29.8 for 31.5) but
// leaves shorter chunks worse dealt (mixed 70 for 50).
template <int D>
struct Geo;
template <>
struct Geo<64> {
  static constexpr int kBlocks = 3, kRingBytes = 48 * 1024;
};
template <>
struct Geo<128> {
  static constexpr int kBlocks = 2, kRingBytes = 64 * 1024;
};

// kLift: a row's bound is put this many powers of two under the largest score that set it, so
// its largest weight is 2^kLift or more there (and 2^(kLift + 8) at most, see weigh). fp16 has
// places of 2^-24 and none below: at 0 the weights of a context's many small keys beside a
// few large ones came out as 0 or 41 % over (16384 keys at 2^-24.5 of the largest).
template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef half8 type;
  static constexpr float kLift = 7.0f;
  static __device__ __forceinline__ floatx16 mm(type a, type b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx4 mm16(type a, type b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<__bf16> {
  typedef __bf16 type __attribute__((ext_vector_type(8)));
  static constexpr float kLift = 0.0f;
  static __device__ __forceinline__ floatx16 mm(type a, type b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx4 mm16(type a, type b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <typename T>
using frag_t = typename Frag<T>::type;

// rowsum_selector (mfma_tile.h) in the operand type T.
template <typename T>
__device__ __forceinline__ frag_t<T> ones_selector(int lane) {
  const half8 h = rowsum_selector(lane);
  frag_t<T> s;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = static_cast<T>(static_cast<float>(h[i]));
  return s;
}

// The kernel's arguments where the launch put them. An item reads them anew through a pointer
// that the compiler cannot see through (`anew`): kept in scalar registers for the whole
// kernel, they and what is derived from them went to VGPR lanes and back.
typedef const __attribute__((address_space(4))) AttendPagedParams &ParamsRef;
typedef const __attribute__((address_space(4))) AttendPagedParams *ParamsPtr;
__device__ __forceinline__ ParamsRef anew(ParamsPtr p) {
  asm volatile("" : "+s"(p));
  return *p;
}

// ---- sequences, items and shares ------------------------------------------------

typedef const __attribute__((address_space(4))) int32_t *uniform_ints;  // read with scalar loads
__device__ __forceinline__ uniform_ints uniform_at(const int32_t *p) {
  return (uniform_ints)(reinterpret_cast<uintptr_t>(p));
}

// A sequence's new tokens: packed rows [t0, t0 + n), the first at position p0. n is below 0
// where its bounds fall within the packed rows.
struct Seq {
  int t0, n, p0;
};
template <typename Ints>
__device__ __forceinline__ Seq load_seq(ParamsRef p, Ints bounds, Ints lens, int b) {
  const int lo = bounds[b], hi = bounds[b + 1];
  Seq s;
  s.t0 = min(max(lo, 0), p.tokens);
  s.n = min(max(hi, 0), p.tokens) - s.t0;
  // lens[b] - hi + t0, kept far from overflow whatever the buffers hold.
  const int64_t p0 = static_cast<int64_t>(lens[b]) - hi + s.t0;
  s.p0 = static_cast<int>(min(max(p0, static_cast<int64_t>(-(1 << 30))),
                              static_cast<int64_t>(1 << 30)));
  return s;
}
// Items of a sequence (per K/V head): `count` tiles of `tokens` tokens.
struct Tiles {
  int count, tokens;
  int step;  // borders inside its items lie at multiples of this many key tiles
};
template <bool SCALAR>  // n is the wave's, not the lane's
__device__ __forceinline__ Tiles tiles_of(ParamsRef p, int n) {
  Tiles t;
  const bool narrow = n <= p.narrow_tokens;
  t.tokens = narrow ? max(n, 1) : p.wide_tokens;
  t.step = narrow ? p.narrow_step : kWideStep;
  // n / wide_tokens, rounded up, by its reciprocal (n < 2^24: exact in fp32 to within one).
  int q = static_cast<int>(static_cast<float>(n) * p.wide_inv);
  q += q * p.wide_tokens < n;
  q -= (q - 1) * p.wide_tokens >= n;
  if constexpr (SCALAR) q = __builtin_amdgcn_readfirstlane(q);
  t.count = narrow ? (n > 0 ? 1 : 0) : q;
  return t;
}
// Keys the last token of a tile sees.
__device__ __forceinline__ int key_end(ParamsRef p, const Seq &s, const Tiles &t,
                                       int tile) {
  // p0 + n <= 2^30 + 2^24
  return min(max(s.p0 + min(s.n, (tile + 1) * t.tokens), 0), p.capacity);
}
// Keys that tiles [0, tile) of one K/V head see (taken as if the last tile were whole), in
// units of 2^unit. The host picks the unit that keeps a batch's weight within 30 bits (one
// key, but for batches of 10^9 keys and more).
__device__ __forceinline__ int keys_before(ParamsRef p, const Seq &s,
                                           const Tiles &t, int tile) {
  const int each = min(max(s.p0, 0), p.capacity);
  const int64_t keys = static_cast<int64_t>(tile) * each +
                       (static_cast<int64_t>(tile) * (tile + 1) >> 1) * t.tokens;
  return static_cast<int>(keys >> p.unit);
}
// Weight of those tiles: their keys and `item` units for each.
__device__ __forceinline__ int weight_before(ParamsRef p, const Seq &s,
                                             const Tiles &t, int item, int tile) {
  return tile * item + keys_before(p, s, t, tile);
}

// Key tiles of an item.
__device__ __forceinline__ int key_tiles(int end) { return (end + kTileKeys - 1) / kTileKeys; }

// a / b for 0 <= a < 2^31, 0 < b, quotients below 2^20: a product in fp32, off by at
// most one, corrected. (64-bit integer divisions took 2 us at the start of every block.)
__device__ __forceinline__ int floor_div(int a, int b) {
  int q = static_cast<int>(static_cast<float>(a) * __builtin_amdgcn_rcpf(static_cast<float>(b)));
  const int64_t r = a - static_cast<int64_t>(q) * b;
  return q + (r >= b ? 1 : r < 0 ? -1 : 0);
}

// A share's border: before key tile `kt` of item (b, kvh, tile); `from` is the weight
// of the sequences before b.
struct Border {
  int b, kvh, tile, kt;
  Seq s;
  int from;
};

// The border at weight `at` inside sequence b (0 <= at - from < H_kv * whole).
__device__ __forceinline__ void place_border(ParamsRef p, const Tiles &t, int item,
                                             int at, Border &r) {
  const int whole = weight_before(p, r.s, t, item, t.count);
  at -= r.from;
  r.kvh = floor_div(at, whole);
  at -= r.kvh * whole;
  int lo = 0, hi = t.count;  // the last tile whose weight_before is <= at
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (weight_before(p, r.s, t, item, mid) <= at) lo = mid;
    else hi = mid;
  }
  r.tile = lo;
  const int tiles = key_tiles(key_end(p, r.s, t, lo));
  const int in = max(at - weight_before(p, r.s, t, item, lo) - item, 0);
  r.kt = static_cast<int>(min((static_cast<int64_t>(in) << p.unit) / kTileKeys,
                              static_cast<int64_t>(tiles)));
  r.kt -= r.kt % t.step;
  // A border close to an item's end moves there, and none cuts a short item: a partial
  // costs more than the keys it balances.
  if (tiles <= kWholeSteps * t.step) r.kt = 0;
  else if (r.kt > tiles - t.step) r.kt = tiles;
}

// The shares that an item of `tiles` key tiles at weights [x0, x1) is cut into: the
// first border inside it and the number of pieces. Piece i is share
// first + i - 1's; a border k lies inside when place_border gives it 0 < kt < tiles.
struct Pieces {
  int first, count;
};
// The workspace slot of a piece: a share may end one item and begin the next.
__device__ __forceinline__ int piece_slot(const Pieces &pc, int piece) {
  return 2 * (pc.first + piece - 1) + (piece == 0 ? 1 : 0);
}
__device__ __forceinline__ int ceil_units(ParamsRef p, int64_t keys) {
  return static_cast<int>((keys + (int64_t{1} << p.unit) - 1) >> p.unit);
}
__device__ __forceinline__ Pieces pieces_of(ParamsRef p, const Tiles &t,
                                            int item, int x0, int x1, int tiles, int share) {
  Pieces r;
  asm volatile("" : "+s"(share));  // its reciprocal is taken here, not kept from the prologue
  const int start = x0 + item + ceil_units(p, t.step * kTileKeys);
  r.first = __builtin_amdgcn_readfirstlane(floor_div(start + share - 1, share));
  const int64_t beyond = tiles - tiles % t.step;
  const int stop = min(x1, x0 + item + ceil_units(p, beyond * kTileKeys));
  r.count = __builtin_amdgcn_readfirstlane(floor_div(stop + share - 1, share)) - r.first + 1;
  return r;
}

// The first sequence behind b that has tokens, or p.batch, 64 at a time: batches that keep
// a slot per user hold runs of empty ones (one token in every 8 of 256 slots 11.4 -> 9.4 us
// against one by one, 2 of 1024: 198 -> 15).
__device__ __forceinline__ int next_filled(ParamsRef p, int b) {
  for (++b; b < p.batch; b += kWave) {
    const int at = b + fresh_lane();
    const bool filled = at < p.batch && load_seq(p, p.cu_tokens, p.seq_lens, at).n > 0;
    const uint64_t found = __builtin_amdgcn_ballot_w64(filled);
    if (found != 0) return b + __builtin_ctzll(found);
  }
  return p.batch;
}

// Inclusive sum over the wave's lanes (DPP row shifts and broadcasts).
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15, rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31, rows 2 and 3
  return x;
}

// A V^T operand from two transposed reads (four keys each) of a V tile.
template <typename T>
__device__ __forceinline__ frag_t<T> read_v(unsigned tile, int first, int second) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4v lds_short4;
  auto read = [&](int off) {
    return __builtin_bit_cast(t4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<lds_short4 *>(static_cast<uintptr_t>(tile + 2u * off))));
  };
  const t4 a = read(first), b = read(second);
  return frag_t<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// ---- a wave's rows -----------------------------------------------------------------

template <typename T, int D>
struct Rows {
  frag_t<T> q[D / 16];   // Q^T fragments: query l % 32 of the wave's rows
  floatx16 o[D / 32];    // O^T accumulators
  floatx4 l;             // row sum (element 0), of the rounded weights
  float m;               // the bound the weights are taken against (log2 units)
  int pos;               // position of the lane's query
};

template <typename T, int D>
__device__ __forceinline__ void clear_rows(Rows<T, D> &r) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int a = 0; a < 16; ++a) r.o[i][a] = 0.f;
#pragma unroll
  for (int a = 0; a < 4; ++a) r.l[a] = 0.f;
  r.m = -INFINITY;
}

// row / group for row < 128, by the host's ceil(2^16 / group): exact, the product is over
// by less than 128 / 2^16 < 1 / group.
__device__ __forceinline__ int token_of(ParamsRef p, int row) {
  return (row * p.group_inv) >> 16;
}

struct Item {
  int t0, n, p0;     // packed tokens and the first one's position
  int kvh;
  int kt0, kt1;      // key tiles of this share
  int end, last;     // keys the item sees (the last token's), and the last one (0 without any)
  int slot;          // partial slot, -1: the whole item
  int wave;          // the calling wave's index in its block
  uniform_ints table;
  const char *k, *v;  // the K/V head's rows of page 0
};

// An item's query row, and its position.
template <typename T>
__device__ __forceinline__ const T *query_row(ParamsRef p, const Item &it, int row,
                                              int &pos) {
  const int token = token_of(p, row);
  const int head = it.kvh * p.group + row - token * p.group;
  pos = it.p0 + token;
  return static_cast<const T *>(p.q) + static_cast<int64_t>(it.t0 + token) * p.q_token +
         static_cast<int64_t>(head) * p.q_head;
}
template <typename T>
__device__ __forceinline__ frag_t<T> load_query(ParamsRef p, const T *q) {
  const unsigned flip = p.negate ? 0x80008000u : 0u;  // a negative scale: -q, exactly
  uint4 x = *reinterpret_cast<const uint4 *>(q);
  x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
  return __builtin_bit_cast(frag_t<T>, x);
}

// ---- one tile of KB 32-key blocks: scores, softmax, products ------------------------

// A 16-byte operand of an LDS tile, `off` halves (per lane) from its byte address.
template <typename T>
__device__ __forceinline__ frag_t<T> read_frag(unsigned tile, int off) {
  typedef __attribute__((address_space(3))) const frag_t<T> lds_frag;
  return *reinterpret_cast<lds_frag *>(static_cast<uintptr_t>(tile + 2u * off));
}

// The reads of a tile's K operands run ahead of the products, as the compiler schedules them:
// with addresses that it could not move a read past, each product waited for its own
// read (long chunks of head_dim 128 515 us for 482).
template <typename T, int D, int KB>
__device__ __forceinline__ void scores(unsigned tile, const FragOffsetsD<D> &fo,
                                       const Rows<T, D> &r, floatx16 (&s)[KB]) {
  frag_t<T> k[D / 16][KB];
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) k[i][kb] = read_frag<T>(tile, fo.k[i] + kb * 32 * D);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a) s[kb][a] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = Frag<T>::mm(k[i][kb], r.q[i], s[kb]);
}

// All of a tile's V^T operands. (Read before the softmax, to land under it: no faster, with
// every register taken.)
template <typename T, int D, int KB>
struct ValueFrags {
  frag_t<T> f[D / 32][2 * KB];
};
template <typename T, int D, int KB>
__device__ __forceinline__ void read_values(unsigned tile, const FragOffsetsD<D> &fo,
                                            ValueFrags<T, D, KB> &v) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int ks = 0; ks < 2 * KB; ++ks)
      v.f[db][ks] = read_v<T>(tile, fo.v[db] + ks * 16 * D, fo.v[db] + (ks * 16 + 8) * D);
}

// Hides keys above `lim` (the lane's position less the tile's first key and the
// lane half's row offset) and those of absent pages (bit i of `absent`: rows
// [16 i, +16) of the tile).
template <int KB>
__device__ __forceinline__ void hide(floatx16 (&s)[KB], int lim, unsigned absent) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a) {
      const bool gone = (absent >> (2 * kb + (a >> 3))) & 1;
      s[kb][a] = (kb * 32 + 8 * (a >> 2) + (a & 3) <= lim && !gone) ? s[kb][a] : -INFINITY;
    }
}

// Weights of the tile as P^T fragments. The bound m moves only when a row's scores pass the one
// that set it by more than 2^8 (weights up to 2^(kLift + 8) fit either type): O is rescaled a
// few times per item instead of per tile.
template <typename T, int D, int KB>
__device__ __forceinline__ void weigh(floatx16 (&s)[KB], float c, Rows<T, D> &r,
                                      frag_t<T> (&w)[2 * KB]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a) mx = fmaxf(mx, s[kb][a]);
  mx = max_lane_pair(mx) * c - Frag<T>::kLift;
  if (__builtin_amdgcn_ballot_w64(mx > r.m + 8.0f) != 0) {
    const float m = fmaxf(r.m, mx);
    const float alpha = m == -INFINITY ? 1.0f : fast_exp2(r.m - m);
    r.m = m;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int a = 0; a < 16; ++a) r.o[i][a] *= alpha;
    r.l[0] *= alpha;
  }
  const float m = r.m == -INFINITY ? 0.0f : r.m;  // a row that has seen no key yet
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a)
      w[2 * kb + (a >> 3)][a & 7] = static_cast<T>(fast_exp2(__builtin_fmaf(s[kb][a], c, -m)));
}

template <typename T, int D, int KB>
__device__ __forceinline__ void accumulate(const ValueFrags<T, D, KB> &v, const frag_t<T> &ones,
                                           const frag_t<T> (&w)[2 * KB], Rows<T, D> &r) {
#pragma unroll
  for (int ks = 0; ks < 2 * KB; ++ks) {
    r.l = Frag<T>::mm16(ones, w[ks], r.l);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) r.o[db] = Frag<T>::mm(v.f[db][ks], w[ks], r.o[db]);
  }
}

// x[l] + x[l ^ 32], and x[l] + x[l ^ 16] + x[l ^ 32] + x[l ^ 48], for every lane (VALU only,
// asm as in max_lane_pair, mfma_tile.h).
__device__ __forceinline__ float sum_lane_pair(float x) {
  float a = x, b = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 0\n\tv_add_f32 %0, %0, %1"
               : "+v"(a), "+v"(b));
  return a;
}
__device__ __forceinline__ float sum_lane_groups(float x) {
  float a = sum_lane_pair(x), b = a;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 0\n\tv_add_f32 %0, %0, %1"
               : "+v"(a), "+v"(b));
  return a;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// `x` with the keys past `lim` cleared. Element e is key offset STRIDE (e / 4) + e % 4 from
// the lane's first. (By bit masks: 8 compares per operand would need more scalar registers
// than there are.)
template <typename T, int STRIDE>
__device__ __forceinline__ frag_t<T> keys_up_to(const frag_t<T> &x, int lim) {
  uint4 b = __builtin_bit_cast(uint4, x);
  auto keep = [lim](unsigned bits, int key) {  // elements `key` and `key` + 1
    const int low = (key - 1 - lim) >> 31, high = (key - lim) >> 31;
    return bits & static_cast<unsigned>((low & 0xffff) | (high & ~0xffff));
  };
  b.x = keep(b.x, 0);
  b.y = keep(b.y, 2);
  b.z = keep(b.z, STRIDE);
  b.w = keep(b.w, STRIDE + 2);
  return __builtin_bit_cast(frag_t<T>, b);
}

// accumulate for rows that must not meet what they do not see (careful passes). The sum of
// the weights is taken lane by lane: the selector of the fast pass multiplies the weights
// of the query 16 columns on by zero, so a NaN there would reach this row. In a masked
// tile (`seen`) the products run once per position among the wave's rows, with the keys
// past that position cleared, and the rows there take the result.
template <typename T, int D, int KB>
__device__ __forceinline__ void accumulate_seen(unsigned tile, const FragOffsetsD<D> &fo,
                                                const frag_t<T> (&w)[2 * KB], bool seen,
                                                int first_key, Rows<T, D> &r) {
  float sum = 0.f;
#pragma unroll
  for (int ks = 0; ks < 2 * KB; ++ks)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += static_cast<float>(w[ks][e]);
  r.l[0] += sum_lane_pair(sum);
#pragma unroll 1
  for (uint64_t todo = ~uint64_t{0}; todo != 0;) {
    const int pos = seen ? __builtin_amdgcn_readlane(r.pos, __builtin_ctzll(todo)) : 0x7fffffff;
    todo &= seen ? ~__builtin_amdgcn_ballot_w64(r.pos == pos) : 0;
#pragma unroll
    for (int ks = 0; ks < 2 * KB; ++ks) {
      const int lim = pos - first_key - 16 * ks;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        const frag_t<T> v = keys_up_to<T, 8>(
            read_v<T>(tile, fo.v[db] + ks * 16 * D, fo.v[db] + (ks * 16 + 8) * D), lim);
        const floatx16 o = Frag<T>::mm(v, w[ks], r.o[db]);
#pragma unroll
        for (int a = 0; a < 16; ++a) r.o[db][a] = r.pos == pos || !seen ? o[a] : r.o[db][a];
        __builtin_amdgcn_sched_barrier(0);  // one operand at a time: this path is rare
      }
    }
  }
}

// ---- pages --------------------------------------------------------------------------

// Page ids of the N 16-key slabs from `key` on: N scalar loads, in flight together. Keys
// past the end lie on no page of their own: the last key's page stands in (the first page of
// an item without keys, which loads nothing).
template <int N>
struct PageIds {
  int id[N];
};
template <int N>
__device__ __forceinline__ PageIds<N> page_ids(ParamsRef p, const Item &it,
                                               int key) {
  PageIds<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i)
    r.id[i] = it.table[min(key + 16 * i, it.last) >> p.page_shift];
  return r;
}
__device__ __forceinline__ bool is_absent(ParamsRef p, int id) {
  return static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_pages);
}
// Bit i: slab i lies on a page outside the pool.
template <int N>
__device__ __forceinline__ unsigned absent_of(ParamsRef p, const PageIds<N> &ids) {
  unsigned absent = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) absent |= is_absent(p, ids.id[i]) ? 1u << i : 0u;
  return absent;
}
// Byte offsets, from the K/V head's rows of page 0, of the 16 keys from `key` + 16 i on, which
// lie in one page; page 0 stands in for one outside the pool. K and V share them.
template <int N>
struct Slabs {
  uint64_t at[N];
};
template <int D, int N>
__device__ __forceinline__ Slabs<N> slabs_of(ParamsRef p, const Item &it,
                                             const PageIds<N> &ids, int key) {
  Slabs<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned page = is_absent(p, ids.id[i]) ? 0u : static_cast<unsigned>(ids.id[i]);
    const unsigned row = static_cast<unsigned>(key + 16 * i) & ((1u << p.page_shift) - 1);
    r.at[i] = static_cast<uint64_t>(page) * p.page_bytes + row * (D * 2);
  }
  return r;
}

// Per-lane source offsets (bytes) of the 16-byte pieces that fill 16 rows of a K or V
// tile: load instruction j writes 1 KiB of LDS, 64 / (D / 8) rows, and adds 1024 j itself.
template <int D, bool NARROW>
struct LoadOffsets {
  unsigned k[D / 32], v[D / 32];
};
template <int D, bool NARROW>
__device__ __forceinline__ LoadOffsets<D, NARROW> load_offsets(int lane) {
  LoadOffsets<D, NARROW> lo;
  constexpr int kChunks = D / 8;
  const int chunk = lane % kChunks, row0 = lane / kChunks;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const int row = j * (64 / kChunks) + row0;
    const int v_swz = NARROW ? group_v_swz<D>(row) : v_swz_d<D>(row);
    lo.k[j] = static_cast<unsigned>(row0 * D + ((chunk ^ k_swz_d<D>(row)) << 3)) * 2;
    lo.v[j] = static_cast<unsigned>(row0 * D + ((chunk ^ v_swz) << 3)) * 2;
  }
  return lo;
}
// The loads of one slab: m0 is set once, each instruction's offset counts for the global
// and for the LDS address (global_to_lds16 in mfma_tile.h says why this is asm).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int D, bool ONCE>
__device__ __forceinline__ void load_slab(const char *base, const unsigned (&off)[D / 32],
                                          unsigned lds) {
  const unsigned m0 = __builtin_amdgcn_readfirstlane(lds);
  if constexpr (D == 64 && ONCE)
    asm volatile(
        "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2 nt\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:1024 nt"
        ::"v"(off[0]), "v"(off[1]), "s"(base), "s"(m0) : "memory", "m0");
  else if constexpr (D == 64)
    asm volatile(
        "s_mov_b32 m0, %3\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:1024"
        ::"v"(off[0]), "v"(off[1]), "s"(base), "s"(m0) : "memory", "m0");
  else if constexpr (ONCE)
    asm volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %4 nt\n\t"
        "global_load_lds_dwordx4 %1, %4 offset:1024 nt\n\t"
        "global_load_lds_dwordx4 %2, %4 offset:2048 nt\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:3*1024 nt"
        ::"v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(m0)
        : "memory", "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %4\n\t"
        "global_load_lds_dwordx4 %1, %4 offset:1024\n\t"
        "global_load_lds_dwordx4 %2, %4 offset:2048\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:3*1024"
        ::"v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base), "s"(m0)
        : "memory", "m0");
}
#pragma clang diagnostic pop

// ---- results -------------------------------------------------------------------------

// Partial of a share. Narrow items: rows of D floats, then (m, l) pairs from slot_rows D
// on. Wide items: each wave's accumulators as (pair of elements, lane), then the pairs.
__device__ __forceinline__ float *partial_of(ParamsRef p, int slot, int head_dim) {
  return p.partials + static_cast<int64_t>(slot) * p.slot_rows * (head_dim + 2);
}

// Two floats of a partial, for another block: coherent 8-byte stores and loads (mfma_tile.h).
// They go past the L2, so the lanes of an instruction must cover contiguous memory: with
// a wide item's rows stored row by row (8 bytes in each of 32 rows per instruction) a
// prompt of 4096 tokens and 14 heads took 85.6 us, in accumulator order 58.6.
typedef float floatx2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void publish2(float *p, float x, float y) {
  const floatx2 a = {x, y};
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p), __builtin_bit_cast(uint64_t, a),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ floatx2 fetch2(const float *p) {
  return __builtin_bit_cast(
      floatx2, __hip_atomic_load(reinterpret_cast<uint64_t *>(const_cast<float *>(p)),
                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <typename T>
__device__ __forceinline__ T *out_row(ParamsRef p, int t0, int kvh, int row,
                                      int head_dim) {
  const int token = token_of(p, row);
  const int head = kvh * p.group + row - token * p.group;
  return static_cast<T *>(p.out) +
         (static_cast<int64_t>(t0 + token) * p.heads + head) * head_dim;
}

template <typename T>
__device__ __forceinline__ void store4(T *dst, const floatx4 &x) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = static_cast<T>(x[i]);
  *reinterpret_cast<t4 *>(dst) = y;
}

// ---- items ----------------------------------------------------------------------------

__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Clears the V rows [from, rows) of a tile, and those of absent pages.
template <int D>
__device__ __forceinline__ void clear_v(unsigned tile, int rows, int from, unsigned absent,
                                        int thread, int threads) {
  typedef __attribute__((address_space(3))) floatx4 lds_floatx4;
  for (int i = thread; i < rows * (D / 8); i += threads) {
    const int row = i / (D / 8);
    if (row >= from || ((absent >> (row / 16)) & 1)) {
      const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<lds_floatx4 *>(static_cast<uintptr_t>(tile + 16u * i)) = zero;
    }
  }
}

// Normalises and stores the lane's half of its query row.
template <typename T, int D>
__device__ __forceinline__ void write_rows(ParamsRef p, const Item &it, int row,
                                           int g, const floatx16 (&o)[D / 32], float l) {
  if (row >= it.n * p.group) return;
  const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;  // NaN stays NaN
  T *out = out_row<T>(p, it.t0, it.kvh, row, D);
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const floatx4 x = {o[i][4 * a] * inv, o[i][4 * a + 1] * inv, o[i][4 * a + 2] * inv,
                         o[i][4 * a + 3] * inv};
      store4<T>(out + 32 * i + 8 * a + 4 * g, x);
    }
}

// One pass over a wide item's keys. Its weights of zero hide no infinity or NaN (0 * inf): the
// CAREFUL pass, which takes about twice as long, runs again over an item that the first
// one left with a result that is not finite.
template <typename T, int D, bool CAREFUL>
__device__ __forceinline__ void wide_pass(ParamsRef p, const Item &it,
                                          unsigned ring, Rows<T, D> &r) {
  constexpr int kTileBytes = kTileKeys * D * 2;
  constexpr int kStages = Geo<D>::kRingBytes / (2 * kTileBytes);
  constexpr int kLoads = 2 * (D / 32);  // a wave's loads per tile
  const int lane = fresh_lane();  // per-lane offsets live in one kind of item only
  const int wave = it.wave;
  const int g = lane >> 5;
  const int rows = it.n * p.group;
  const int row = 32 * wave + (lane & 31);
  const FragOffsetsD<D> fo = frag_offsets_d<D>(lane);
  const LoadOffsets<D, false> lo = load_offsets<D, false>(lane);
  const frag_t<T> ones = ones_selector<T>(lane);
  // Positions of the wave's first and last query.
  const int first_pos = it.p0 + token_of(p, min(32 * wave, rows - 1));
  const int last_pos = it.p0 + token_of(p, min(32 * wave + 31, rows - 1));
  const bool has_rows = 32 * wave < rows;

  // Wave w loads rows [16 w, +16) of each tile's K and V. A tile's page ids are read one
  // step before its loads leave; `absent` queues its masks until it is used.
  struct Ids {
    PageIds<kTileKeys / 16> all;
    PageIds<1> own;
  };
  auto ids_of = [&](int kt) {
    return Ids{page_ids<kTileKeys / 16>(p, it, kt * kTileKeys),
               page_ids<1>(p, it, kt * kTileKeys + 16 * wave)};
  };
  unsigned absent[kStages];
  Ids ids = ids_of(it.kt0);
  auto issue = [&](int kt) {
    const int stage = (kt - it.kt0) % kStages;
    const Slabs<1> slab = slabs_of<D>(p, it, ids.own, kt * kTileKeys + 16 * wave);
    const unsigned at = ring + stage * 2 * kTileBytes + 16 * wave * D * 2;
    load_slab<D, false>(it.k + slab.at[0], lo.k, at);
    load_slab<D, false>(it.v + slab.at[0], lo.v, at + kTileBytes);
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    absent[i] = absent_of(p, ids.all);
    if (it.kt0 + i < it.kt1) issue(it.kt0 + i);
    ids = ids_of(it.kt0 + i + 1);
  }
  const T *q = query_row<T>(p, it, min(row, rows - 1), r.pos);  // rows past the last repeat it
#pragma unroll
  for (int s = 0; s < D / 16; ++s) r.q[s] = load_query<T>(p, q + (D / 2) * g + 8 * s);
  clear_rows<T, D>(r);
  for (int kt = it.kt0; kt < it.kt1; ++kt) {
    // Tile kt has landed once at most the later tiles' loads are outstanding.
    const int later = min(kStages - 2, it.kt1 - 1 - kt);
    if (kStages > 2 && later >= 2) wait_loads<2 * kLoads>();
    else if (kStages > 2 && later == 1) wait_loads<kLoads>();
    else wait_loads<0>();
    block_barrier();
    absent[kStages - 1] = absent_of(p, ids.all);
    if (kt + kStages - 1 < it.kt1) issue(kt + kStages - 1);
    ids = ids_of(kt + kStages);
    const unsigned k_tile = ring + ((kt - it.kt0) % kStages) * 2 * kTileBytes;
    const unsigned v_tile = k_tile + kTileBytes;
    const int key0 = kt * kTileKeys;
    const unsigned gone = absent[0];
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) absent[i] = absent[i + 1];
    if (gone != 0 || key0 + kTileKeys > it.end) {
      clear_v<D>(v_tile, kTileKeys, it.end - key0, gone, 64 * wave + fresh_lane(), kThreads);
      block_barrier();
    }
    if (!has_rows || last_pos < key0) continue;
    floatx16 s[2];
    frag_t<T> weights[4];
    scores<T, D, 2>(k_tile, fo, r, s);
    const bool masked =
        gone != 0 || first_pos < key0 + kTileKeys - 1 || key0 + kTileKeys > it.end;
    if (masked)
      hide<2>(s, min(r.pos, it.end - 1) - key0 - 4 * g, gone);
    weigh<T, D, 2>(s, p.c, r, weights);
    if constexpr (CAREFUL) {
      accumulate_seen<T, D, 2>(v_tile, fo, weights, masked, key0 + 4 * g, r);
    } else {
      ValueFrags<T, D, 2> v;
      read_values<T, D, 2>(v_tile, fo, v);
      accumulate<T, D, 2>(v, ones, weights, r);
    }
  }
  block_barrier();  // the ring may be filled again
}

template <typename T, int D>
__device__ __forceinline__ void wide_item(ParamsRef p, const Item &it,
                                          unsigned ring, int *votes, Rows<T, D> &r) {
  const int wave = it.wave;
  const bool has_rows = 32 * wave < it.n * p.group;
  wide_pass<T, D, false>(p, it, ring, r);
  // Sums of finite values below 2^100 are finite, so one sum tells for all of them.
  float probe = r.l[0];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int a = 0; a < 16; ++a) probe += r.o[i][a];
  const bool lost = __builtin_amdgcn_ballot_w64(has_rows && !is_finite(probe)) != 0;
  if (fresh_lane() == 0) votes[wave] = lost;
  block_barrier();
  if (votes[0] | votes[1] | votes[2] | votes[3]) wide_pass<T, D, true>(p, it, ring, r);
}

// Stores a wave's rows of a wide item as a partial: its accumulators, then (m, l) pairs.
template <typename T, int D>
__device__ __forceinline__ void publish_wide(ParamsRef p, const Item &it, int slot,
                                             const Rows<T, D> &r) {
  const int lane = fresh_lane(), wave = it.wave;
  if (32 * wave >= it.n * p.group) return;
  float *part = partial_of(p, slot, D) + wave * (32 * D) + 2 * lane;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int a = 0; a < 8; ++a)
      publish2(part + (8 * i + a) * 128, r.o[i][2 * a], r.o[i][2 * a + 1]);
  if (lane < 32)
    publish2(partial_of(p, slot, D) + kWideRows * D + 2 * (32 * wave + lane), r.m, r.l[0]);
}

// o a + x b, both products rounded: the same bits whichever of the two came from the
// workspace.
__device__ __forceinline__ float fold(float o, float a, float x, float b) {
#pragma clang fp contract(off)
  return o * a + x * b;
}

// Joins a partial to a wave's rows.
template <typename T, int D>
__device__ __forceinline__ void merge_wide(ParamsRef p, const Item &it, int slot, Rows<T, D> &r) {
  const int lane = fresh_lane(), wave = it.wave;
  if (32 * wave >= it.n * p.group) return;
  const float *part = partial_of(p, slot, D);
  const floatx2 ml = fetch2(part + kWideRows * D + 2 * (32 * wave + (lane & 31)));
  floatx2 x[D / 4];
#pragma unroll
  for (int i = 0; i < D / 4; ++i) x[i] = fetch2(part + wave * (32 * D) + 128 * i + 2 * lane);
  const float top = fmaxf(r.m, ml[0]);
  const float a = r.m == -INFINITY ? 0.f : fast_exp2(r.m - top);
  const float b = ml[0] == -INFINITY ? 0.f : fast_exp2(ml[0] - top);
  r.m = top;
  r.l[0] = fold(r.l[0], a, ml[1], b);
#pragma unroll
  for (int i = 0; i < D / 4; ++i) {
    r.o[i / 8][2 * (i % 8)] = fold(r.o[i / 8][2 * (i % 8)], a, x[i][0], b);
    r.o[i / 8][2 * (i % 8) + 1] = fold(r.o[i / 8][2 * (i % 8) + 1], a, x[i][1], b);
  }
}

// Narrow items run on v_mfma_f32_16x16x32, with NQ groups of 16 query rows: with the
// 32-row products a group of 7 query heads paid for 32 rows of softmax (32 ragged sequences
// of 14/2 heads 16.3 us for 14.5).
// Lane l: query l % 16 of a group, g = l / 16. S^T of 16 keys: A = K rows (k-step s, lane g:
// dims [32 s + 8 g, +8)), B = Q^T alike; the lane gets keys 4 g + j. O^T of 16 dims: A = V^T,
// k index 8 g + 4 part + e standing for key 16 part + 4 g + e of a 32-key step, which is how
// the lane's own weights of two 16-key blocks lie; the lane gets dims 4 g + j.
template <typename T, int D, int NQ>
struct NarrowRows {
  floatx4 o[NQ][D / 16];
  float m[NQ], l[NQ];  // l: the lane's share of the row sum
};

// One pass over the wave's keys of a narrow item; CAREFUL as in wide_pass.
template <typename T, int D, int NQ, bool CAREFUL>
__device__ __forceinline__ void narrow_pass(ParamsRef p, const Item &it,
                                            unsigned ring, NarrowRows<T, D, NQ> &r) {
  constexpr int kKeys = kNarrowKeys;
  constexpr int KB = kKeys / 16;
  constexpr int kTileBytes = kKeys * D * 2;
  constexpr int kLoads = kTileBytes / 1024;  // load instructions per tile
  const int lane = fresh_lane();  // per-lane offsets live in one kind of item only
  const int wave = it.wave;
  const int col = lane & 15, g = lane >> 4;
  const int rows = it.n * p.group;
  const unsigned k_tile = ring + wave * 2 * kTileBytes, v_tile = k_tile + kTileBytes;
  const int stop = min(it.end, it.kt1 * kTileKeys);
  typedef PageIds<kKeys / 16> Ids;
  typedef Slabs<kKeys / 16> WaveSlabs;
  auto issue = [&](const WaveSlabs &slabs, const char *base, const unsigned (&off)[D / 32],
                   unsigned lds) {
#pragma unroll
    for (int i = 0; i < kKeys / 16; ++i)
      load_slab<D, true>(base + slabs.at[i], off, lds + 16 * i * D * 2);
  };
  int key0 = it.kt0 * kTileKeys + wave * kKeys;
  Ids ids = page_ids<kKeys / 16>(p, it, key0);
  const LoadOffsets<D, true> lo = load_offsets<D, true>(lane);
  if (key0 < stop) {
    const WaveSlabs slabs = slabs_of<D>(p, it, ids, key0);
    issue(slabs, it.k, lo.k, k_tile);
    issue(slabs, it.v, lo.v, v_tile);
  }
  frag_t<T> q[NQ][D / 32];
  int pos[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const T *row = query_row<T>(p, it, min(16 * i + col, rows - 1), pos[i]);
#pragma unroll
    for (int s = 0; s < D / 32; ++s) q[i][s] = load_query<T>(p, row + 32 * s + 8 * g);
  }
  // Fragment offsets, in halves: K chunk 4 s + g of row `col`; V rows 4 g + col / 4, dims
  // 16 db + 4 (col % 4).
  int fk[D / 32], fv[D / 16];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) fk[s] = col * D + (((4 * s + g) ^ k_swz_d<D>(col)) << 3);
  const int v_row = 4 * g + (col >> 2);
#pragma unroll
  for (int db = 0; db < D / 16; ++db)
    fv[db] = v_row * D + (((2 * db + ((col >> 1) & 1)) ^ group_v_swz<D>(v_row)) << 3) + 4 * (col & 1);

  auto &o = r.o;
  auto &m = r.m;
  auto &l = r.l;
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[i][db] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  for (; key0 < stop; key0 += kWaves * kKeys) {
    const int next = key0 + kWaves * kKeys;
    const unsigned absent = absent_of(p, ids);
    ids = page_ids<kKeys / 16>(p, it, next);
    // Loads leave in the order K, V, K, V: at most those of V are younger than K's.
    wait_loads<kLoads>();
    floatx4 s[NQ][KB];
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[i][kb] = floatx4{0.f, 0.f, 0.f, 0.f};
    frag_t<T> k[D / 32][KB];
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) k[st][kb] = read_frag<T>(k_tile, fk[st] + kb * 16 * D);
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < NQ; ++i) s[i][kb] = Frag<T>::mm16(k[st][kb], q[i][st], s[i][kb]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read before it is overwritten
    const WaveSlabs slabs = slabs_of<D>(p, it, ids, next);
    if (next < stop) issue(slabs, it.k, lo.k, k_tile);
    const bool masked = absent != 0 || it.p0 < key0 + kKeys - 1 || key0 + kKeys > it.end;
    if (masked) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const int lim = min(pos[i], it.end - 1) - key0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][kb][j] =
                (16 * kb + j <= lim && !((absent >> kb) & 1)) ? s[i][kb][j] : -INFINITY;
      }
    }
    // Weights, split into two parts of the type, and the bound m (as in weigh).
    frag_t<T> hi[NQ][KB / 2], low[NQ][KB / 2];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[i][kb][j]);
      mx = max_lane_groups(mx) * p.c - Frag<T>::kLift;
      if (__builtin_amdgcn_ballot_w64(mx > m[i] + 8.0f) != 0) {
        const float top = fmaxf(m[i], mx);
        const float alpha = top == -INFINITY ? 1.0f : fast_exp2(m[i] - top);
        m[i] = top;
        l[i] *= alpha;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) o[i][db] *= alpha;
      }
      const float bound = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = fast_exp2(__builtin_fmaf(s[i][kb][j], p.c, -bound));
          const T h = static_cast<T>(w);
          hi[i][kb / 2][4 * (kb % 2) + j] = h;
          low[i][kb / 2][4 * (kb % 2) + j] = static_cast<T>(w - static_cast<float>(h));
          l[i] += w;
        }
    }
    if (next < stop) wait_loads<kLoads>();
    else wait_loads<0>();
    if (absent != 0 || key0 + kKeys > it.end) {
      clear_v<D>(v_tile, kKeys, it.end - key0, absent, fresh_lane(), kWave);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (CAREFUL && masked) {
#pragma unroll
      for (int i = 0; i < NQ; ++i)  // as accumulate_seen
#pragma unroll 1
        for (uint64_t todo = ~uint64_t{0}; todo != 0;) {
          const unsigned tile = uniform_lds_u(v_tile);  // no address of this path is hoisted
          const int at = __builtin_amdgcn_readlane(pos[i], __builtin_ctzll(todo));
          todo &= ~__builtin_amdgcn_ballot_w64(pos[i] == at);
#pragma unroll
          for (int db = 0; db < D / 16; ++db) {
            floatx4 x = o[i][db];
#pragma unroll
            for (int ks = 0; ks < KB / 2; ++ks) {
              const frag_t<T> v = keys_up_to<T, 16>(
                  read_v<T>(tile, fv[db] + 32 * ks * D, fv[db] + (32 * ks + 16) * D),
                  at - key0 - 4 * g - 32 * ks);
              x = Frag<T>::mm16(v, hi[i][ks], x);
              x = Frag<T>::mm16(v, low[i][ks], x);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) o[i][db][a] = pos[i] == at ? x[a] : o[i][db][a];
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    } else {
      frag_t<T> v[D / 16][KB / 2];
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int ks = 0; ks < KB / 2; ++ks)
          v[db][ks] = read_v<T>(v_tile, fv[db] + 32 * ks * D, fv[db] + (32 * ks + 16) * D);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int ks = 0; ks < KB / 2; ++ks)
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            o[i][db] = Frag<T>::mm16(v[db][ks], hi[i][ks], o[i][db]);
            o[i][db] = Frag<T>::mm16(v[db][ks], low[i][ks], o[i][db]);
          }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next < stop) issue(slabs, it.v, lo.v, v_tile);
  }
}

template <typename T, int D, int NQ>
__device__ __forceinline__ void narrow_item(ParamsRef p, const Item &it,
                                            unsigned ring, float *exchange, float *exchange_ml) {
  const int rows = it.n * p.group, wave = it.wave;
  NarrowRows<T, D, NQ> r;
  narrow_pass<T, D, NQ, false>(p, it, ring, r);
  // Rows of one token see the same keys: nothing that any of them should not see is left.
  if (rows > p.group) {
    float probe = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      probe += r.l[i];
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a) probe += r.o[i][db][a];
    }
    if (__builtin_amdgcn_ballot_w64(!is_finite(probe)) != 0)
      narrow_pass<T, D, NQ, true>(p, it, ring, r);
  }

  // Join the four waves' states. Row r's dims lie in LDS as 16-byte pieces,
  // piece j at j ^ (r & 15).
  const int lane = fresh_lane(), col = lane & 15, g = lane >> 4;
  block_barrier();  // every wave is done with its tiles
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = 16 * i + col;
    const float sum = sum_lane_groups(r.l[i]);
    if (row < rows) {
      float *x = exchange + (wave * kNarrowRows + row) * D;
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        *reinterpret_cast<floatx4 *>(x + 4 * ((4 * db + g) ^ col)) = r.o[i][db];
      if (g == 0) {
        exchange_ml[2 * (wave * kNarrowRows + row)] = r.m[i];
        exchange_ml[2 * (wave * kNarrowRows + row) + 1] = sum;
      }
    }
  }
  block_barrier();
  for (int i = 64 * wave + lane; i < rows * (D / 2); i += kThreads) {
    const int at = i / (D / 2), pair = i % (D / 2);  // two dims per thread
    float m = -INFINITY, l = 0.f;
    float w[kWaves];
#pragma unroll
    for (int j = 0; j < kWaves; ++j) m = fmaxf(m, exchange_ml[2 * (j * kNarrowRows + at)]);
    floatx2 o = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      const float mj = exchange_ml[2 * (j * kNarrowRows + at)];
      w[j] = mj == -INFINITY ? 0.f : fast_exp2(mj - m);
      l += w[j] * exchange_ml[2 * (j * kNarrowRows + at) + 1];
      const floatx2 x = *reinterpret_cast<const floatx2 *>(
          exchange + (j * kNarrowRows + at) * D + 4 * ((pair >> 1) ^ (at & 15)) + 2 * (pair & 1));
      if (mj != -INFINITY) o += w[j] * x;
    }
    if (it.slot < 0) {
      const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
      typedef T t2 __attribute__((ext_vector_type(2)));
      const t2 y = {static_cast<T>(o[0] * inv), static_cast<T>(o[1] * inv)};
      *reinterpret_cast<t2 *>(out_row<T>(p, it.t0, it.kvh, at, D) + 2 * pair) = y;
    } else {
      float *part = partial_of(p, it.slot, D);
      publish2(part + at * D + 2 * pair, o[0], o[1]);
      if (pair == 0) publish2(part + p.slot_rows * D + 2 * at, m, l);
    }
  }
  block_barrier();  // the exchange may be overwritten
}

// Two dims of a narrow item's row, joined from its partials.
struct JoinedRow {
  float m = -INFINITY, l = 0.f;
  floatx2 o = {0.f, 0.f};

  // Joins the first `fresh` of kDeep partials (the others repeat the last one). One without a
  // key that the row sees has l = 0 and o = 0. None is left out for a weight of zero: a NaN or
  // an infinity that the row does see stays in it (0 * inf), as in an item that is not cut.
  template <int kDeep>
  __device__ __forceinline__ void fold(const floatx2 (&ml)[kDeep], const floatx2 (&x)[kDeep],
                                       int fresh) {
    float top = m;
#pragma unroll
    for (int j = 0; j < kDeep; ++j) top = fmaxf(top, ml[j][0]);
    const float base = top == -INFINITY ? 0.f : top;
    const float old = fast_exp2(m - base);
    m = top;
    l *= old;
    o *= old;
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const float a = fast_exp2(ml[j][0] - base);
      l += j < fresh ? a * ml[j][1] : 0.f;
      o[0] += j < fresh ? a * x[j][0] : 0.f;
      o[1] += j < fresh ? a * x[j][1] : 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void write(T *out) const {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;  // NaN stays NaN
    *reinterpret_cast<t2 *>(out) = t2{static_cast<T>(o[0] * inv), static_cast<T>(o[1] * inv)};
  }
};

// Joins a narrow item's pieces, first to last, and writes its rows. kDeep pieces' loads are
// in flight at a time: 8, but 16 where there are more than 8 pieces (32 ragged sequences
// of up to 9 pieces 14.3 -> 14.0 us, two of 8k keys 16.7 -> 16.3; 16 for all: 15.7 for 15.1).
template <typename T, int D, int kDeep>
__device__ __forceinline__ void join_narrow(ParamsRef p, const Item &it,
                                            const Pieces &pc) {
  const int n = it.n * p.group * (D / 2);
  const int thread = 64 * it.wave + fresh_lane();
  for (int i = thread; i < n; i += kThreads) {
    const int row = i / (D / 2), at = 2 * (i % (D / 2));
    JoinedRow r;
    for (int j0 = 0; j0 < pc.count; j0 += kDeep) {
      floatx2 ml[kDeep], x[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int piece = min(j0 + j, pc.count - 1);
        const float *part = partial_of(p, piece_slot(pc, piece), D);
        ml[j] = fetch2(part + p.slot_rows * D + 2 * row);
        x[j] = fetch2(part + row * D + at);
      }
      r.fold(ml, x, pc.count - j0);
    }
    r.write<T>(out_row<T>(p, it.t0, it.kvh, row, D) + at);
  }
}

// Partials of a narrow item to join: partial j lies in slot `at` + j `step`, but the first in
// `at0` and the last in `at1`.
struct NarrowJoin {
  int count, at, step, at0, at1;
};
// Where the join of pieces [16 group, + 16) goes: to the second slot of a share that lies
// within the item and so has no use for it, its first piece's, or its second one's where
// that piece starts the item. A last group of one piece stays in that piece's slot.
__device__ __forceinline__ int group_slot(const Pieces &pc, int group) {
  return group == 0 ? 2 * pc.first + 1
                    : 2 * (pc.first + 16 * group - 1) + (16 * group + 1 < pc.count ? 1 : 0);
}

// Joins them, in order, into slot `dest`, or into the output rows (dest < 0). A function of
// its own beside join_narrow: one for both cost items of few pieces (32 ragged sequences
// 15.0 us for 14.1).
template <typename T, int D>
__device__ __forceinline__ void join_many(ParamsRef p, const Item &it, const NarrowJoin &join,
                                            int dest) {
  constexpr int kDeep = 16;
  int zero;  // per lane, so that the slots' addresses are not scalar: there are too many
  asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
  const int n = it.n * p.group * (D / 2), count = join.count;
  const int thread = 64 * it.wave + fresh_lane();
  for (int i = thread; i < n; i += kThreads) {
    const int row = i / (D / 2), at = 2 * (i % (D / 2));
    JoinedRow r;
    for (int j0 = 0; j0 < count; j0 += kDeep) {
      floatx2 ml[kDeep], x[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int at_j = min(j0 + j, count - 1);
        const int slot = at_j == 0 ? join.at0 : at_j == count - 1 ? join.at1
                                                                  : join.at + at_j * join.step;
        const float *part = partial_of(p, slot + zero, D);
        ml[j] = fetch2(part + p.slot_rows * D + 2 * row);
        x[j] = fetch2(part + row * D + at);
      }
      r.fold(ml, x, count - j0);
    }
    if (dest >= 0) {
      float *part = partial_of(p, dest, D);
      publish2(part + row * D + at, r.o[0], r.o[1]);
      if (at == 0) publish2(part + p.slot_rows * D + 2 * row, r.m, r.l);
      continue;
    }
    r.write<T>(out_row<T>(p, it.t0, it.kvh, row, D) + at);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, Geo<D>::kBlocks) void attend_paged_kernel(const AttendPagedParams) {
  __shared__ __align__(1024) unsigned char ring_mem[Geo<D>::kRingBytes];
  __shared__ __align__(16) float ml_mem[2 * kWaves * kNarrowRows];
  __shared__ int arrived, votes[kWaves];

  const ParamsPtr params = (ParamsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  ParamsRef p = *params;
  // One word of each 64-byte line of the arguments, read together: the lines' misses
  // (their first use in a launch) overlap instead of following one another.
  {
    const auto *args = (uniform_ints)__builtin_amdgcn_kernarg_segment_ptr();
    int touched = 0;
#pragma unroll
    for (unsigned i = 0; i < sizeof(AttendPagedParams); i += 64) touched ^= args[i / 4];
    asm volatile("" ::"s"(touched));
  }
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int n_blocks = static_cast<int>(gridDim.x);
  const uniform_ints bounds = uniform_at(p.cu_tokens), lens = uniform_at(p.seq_lens);
  // Packed rows that belong to no sequence: [0, head) and [tail, tokens).
  const int head = min(max(bounds[0], 0), p.tokens);
  const int last_bound = min(max(bounds[p.batch], 0), p.tokens);

  // Every wave sums the sequences' weights (lane l takes `per` of them) and finds its
  // block's two borders: no exchange between waves, and scalar code from there on.
  const int per = (p.batch + kWave - 1) / kWave;
  int mine = 0, my_items = 0, signs = 0;
  Seq s = {0, 0, 0};
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b >= p.batch) break;
    s = load_seq(p, p.cu_tokens, p.seq_lens, b);
    const Tiles t = tiles_of<false>(p, s.n);
    mine += keys_before(p, s, t, t.count) * p.kv_heads;
    my_items += t.count * p.kv_heads;
    signs |= s.n;
  }
  const int keys_upto = wave_prefix(mine), items_upto = wave_prefix(my_items);
  // Bounds that go up and down can claim a row twice, or more rows than there are, beyond what
  // the weights' 30 bits were chosen for: such a batch has no sequences, and its outputs are zero.
  const bool sound = __builtin_amdgcn_ballot_w64(signs < 0) == 0;
  const int tail = sound ? last_bound : 0;
  const int all_keys = __builtin_amdgcn_readlane(keys_upto, kWave - 1);
  const int all_items = __builtin_amdgcn_readlane(items_upto, kWave - 1);
  const int few = 1 + (kFewItemKeys >> p.unit);
  const int item = __builtin_amdgcn_readfirstlane(
      all_items <= n_blocks && all_keys + all_items * few <= n_blocks * few
          ? few : 1 + (kItemKeys >> p.unit));
  const int total = all_keys + all_items * item;
  mine += my_items * item;
  const int upto = keys_upto + items_upto * item;
  // share * n_blocks > total, whatever the reciprocal's last bit.
  const int share = max(static_cast<int>(__umulhi(total, p.blocks_inv)) + 2, p.min_share);
  // Neighbouring shares read the same keys, so they go to one XCD (blocks are
  // dealt to the 8 XCDs in turn). Any estimate of the shares in use is right here.
  const int active = static_cast<int>(static_cast<float>(total) *
                                      __builtin_amdgcn_rcpf(static_cast<float>(share))) + 1;
  const int per_xcd =
      (__builtin_amdgcn_readfirstlane(min(active, n_blocks)) + 7) / 8;
  const int blk = static_cast<int>(blockIdx.x);
  const int w = blk < 8 * per_xcd && 8 * per_xcd <= n_blocks ? (blk & 7) * per_xcd + (blk >> 3) : blk;
  // Even lanes compute the share's first border, odd lanes its end, in one pass.
  const int at0 = w * share, at1 = at0 + share;
  const int owner0 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= at0));
  const int owner1 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= at1));
  const int owner = (lane & 1) ? owner1 : owner0;
  const int at = (lane & 1) ? at1 : at0;
  Border border;
  border.from = __shfl(upto - mine, owner & 63);
  border.b = owner * per;
  if (per == 1) {
    border.s.t0 = __shfl(s.t0, owner & 63);
    border.s.n = __shfl(s.n, owner & 63);
    border.s.p0 = __shfl(s.p0, owner & 63);
  } else if (sound && owner < kWave) {
    for (;; ++border.b) {  // the owner's sequences
      border.s = load_seq(p, p.cu_tokens, p.seq_lens, border.b);
      const Tiles t = tiles_of<false>(p, border.s.n);
      const int weight = weight_before(p, border.s, t, item, t.count) * p.kv_heads;
      if (at < border.from + weight || border.b + 1 >= p.batch) break;
      border.from += weight;
    }
  }
  if (sound && owner < kWave) place_border(p, tiles_of<false>(p, border.s.n), item, at, border);
  else border.b = p.batch;
  struct { int b, kvh, tile, kt; } end;
  int b = __builtin_amdgcn_readlane(border.b, 0), kvh = __builtin_amdgcn_readlane(border.kvh, 0);
  int tile = __builtin_amdgcn_readlane(border.tile, 0), kt = __builtin_amdgcn_readlane(border.kt, 0);
  int from = __builtin_amdgcn_readlane(border.from, 0);
  s.t0 = __builtin_amdgcn_readlane(border.s.t0, 0);
  s.n = __builtin_amdgcn_readlane(border.s.n, 0);
  s.p0 = __builtin_amdgcn_readlane(border.s.p0, 0);
  end.b = __builtin_amdgcn_readlane(border.b, 1);
  end.kvh = __builtin_amdgcn_readlane(border.kvh, 1);
  end.tile = __builtin_amdgcn_readlane(border.tile, 1);
  end.kt = __builtin_amdgcn_readlane(border.kt, 1);

  const unsigned ring = lds_addr(ring_mem);
  const int all_weight = __builtin_amdgcn_readfirstlane(total);
  Tiles t = tiles_of<true>(p, s.n);
  while (sound && b < p.batch) {
    if (tile >= t.count) {  // next K/V head or sequence
      tile = 0;
      kt = 0;
      if (t.count == 0 || ++kvh >= p.kv_heads) {
        from += weight_before(p, s, t, item, t.count) * p.kv_heads;
        kvh = 0;
        // Nothing but empty sequences follows the last weight.
        b = __builtin_amdgcn_readfirstlane(from) >= all_weight ? p.batch : b + 1;
        if (b >= p.batch) break;
        s = load_seq(p, bounds, lens, b);
        if (s.n == 0) {
          b = __builtin_amdgcn_readfirstlane(next_filled(anew(params), b));
          if (b >= p.batch) break;
          s = load_seq(p, bounds, lens, b);
        }
        t = tiles_of<true>(p, s.n);
      }
      if (b > end.b) break;
      continue;
    }
    const bool last = b == end.b && kvh == end.kvh && tile == end.tile;
    Item it;
    it.end = key_end(p, s, t, tile);
    it.last = __builtin_amdgcn_readfirstlane(max(it.end - 1, 0));
    const int tiles = key_tiles(it.end);
    it.kt0 = kt;
    it.kt1 = last ? min(end.kt, tiles) : tiles;
    it.t0 = s.t0 + tile * t.tokens;
    it.n = min(t.tokens, s.n - tile * t.tokens);
    it.p0 = s.p0 + tile * t.tokens;
    it.kvh = kvh;
    it.wave = wave;
    const uint64_t head_at = static_cast<uint64_t>(kvh) * p.head_bytes;
    it.k = static_cast<const char *>(p.k_pages) + head_at;
    it.v = static_cast<const char *>(p.v_pages) + head_at;
    it.table = uniform_at(p.page_table + static_cast<int64_t>(b) * p.max_pages);
    // A whole item (also one that sees no key) is written out; a part leaves a partial.
    const bool whole = it.kt0 == 0 && it.kt1 == tiles && !(last && end.kt < tiles) &&
                       !(last && tiles == 0);
    if (whole || it.kt1 > it.kt0) {
      it.slot = whole ? -1 : 2 * w + (it.kt0 == 0 ? 1 : 0);
      Pieces pc;
      auto find_pieces = [&] {
        const int x0 = from + kvh * weight_before(p, s, t, item, t.count) +
                       weight_before(p, s, t, item, tile);
        const int x1 = x0 + weight_before(p, s, t, item, tile + 1) - weight_before(p, s, t, item, tile);
        pc = pieces_of(p, t, item, x0, x1, key_tiles(it.end), share);
      };
      // Counts the block at a border (what it stored before is visible first) and returns
      // how many have been there; the `of`-th sets the counter back to zero for the next call.
      auto count_at = [&](int border, int of) {
        wait_loads<0>();
        __syncthreads();
        if (wave == 0 && fresh_lane() == 0) {
          unsigned *counter = p.counters + border;
          arrived = 1 + static_cast<int>(__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                                                __HIP_MEMORY_SCOPE_AGENT));
          if (arrived == of)
            __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        return arrived;
      };
      if (it.n * p.group <= kNarrowRows) {
        float *exchange = reinterpret_cast<float *>(ring_mem);
        if (it.n * p.group <= 16) narrow_item<T, D, 1>(anew(params), it, ring, exchange, ml_mem);
        else narrow_item<T, D, 2>(anew(params), it, ring, exchange, ml_mem);
        if (it.slot >= 0) find_pieces();
        if (it.slot >= 0 && pc.count <= kFlatPieces) {
          if (count_at(pc.first, pc.count) == pc.count) {
            if (pc.count <= 8) join_narrow<T, D, 8>(anew(params), it, pc);
            else join_narrow<T, D, 16>(anew(params), it, pc);
          }
        } else if (it.slot >= 0) {
          // Groups of 16 pieces first, each counted at the border behind its first piece,
          // then the groups.
          const int group = (w - pc.first + 1) / 16;
          NarrowJoin join;
          join.count = min(pc.count - 16 * group, 16);
          join.at0 = piece_slot(pc, 16 * group);
          join.at = 2 * (pc.first + 16 * group - 1);
          join.step = 2;
          join.at1 = join.at + 2 * (join.count - 1);
          int border = pc.first + 16 * group;
          for (;;) {
            const bool whole_item = join.step == 32;
            if (join.count > 1) {
              if (count_at(border, join.count) != join.count) break;
              const int dest = whole_item ? -1 : group_slot(pc, group);
              join_many<T, D>(anew(params), it, join, dest);
              __syncthreads();  // `arrived` may be written again
            }
            if (whole_item) break;
            join.count = (pc.count + 15) / 16;
            join.at0 = group_slot(pc, 0);
            join.at = 2 * (pc.first - 1) + 1;
            join.step = 32;
            join.at1 = group_slot(pc, join.count - 1);
            border = pc.first + 15;
          }
        }
      } else {
        Rows<T, D> r;
        wide_item<T, D>(anew(params), it, ring, votes, r);
        // A cut item's pieces are joined in pairs, the pairs in pairs and so on, by the block
        // of a pair that is there last: a fixed tree, so the order of arrival changes no
        // bit. The other has left its rows in the slot of its first piece. Each pair counts
        // at a border of its own, between its halves; a block that finds the other half
        // there need not store its own. (All pieces by the last block, one by one, at ~2
        // thousand cycles each: 16000 keys and 32 tokens of 14/2 heads 35.4 us for 26.7, 24
        // sequences with 3 chunks 49.4 for 47.4, one token alike.)
        bool holds = true;
        if (it.slot >= 0) find_pieces();
        else pc.count = 1;
        for (int half = 1; half < pc.count; half *= 2) {
          const int mine_from = (w - pc.first + 1) & -half, other = mine_from ^ half;
          if (other >= pc.count) continue;
          const int border = pc.first + max(mine_from, other) - 1;
          __syncthreads();  // `arrived` has been read
          if (wave == 0 && fresh_lane() == 0) {
            unsigned *counter = p.counters + border;
            arrived = static_cast<int>(__hip_atomic_load(counter, __ATOMIC_RELAXED,
                                                         __HIP_MEMORY_SCOPE_AGENT));
            if (arrived != 0)
              __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
          __syncthreads();
          if (arrived == 0) {
            publish_wide<T, D>(anew(params), it, piece_slot(pc, mine_from), r);
            if (count_at(border, 2) == 1) {
              holds = false;
              break;
            }
          }
          merge_wide<T, D>(anew(params), it, piece_slot(pc, other), r);
        }
        if (holds && 32 * wave < it.n * p.group) {
          const int lane = fresh_lane();
          write_rows<T, D>(anew(params), it, 32 * wave + (lane & 31), lane >> 5, r.o, r.l[0]);
        }
      }
      if (it.slot >= 0) __syncthreads();  // `arrived` may be written again
    }
    if (last) break;
    ++tile;
    kt = 0;
  }

  // Outputs of packed rows that belong to no sequence are zero.
  if (sound && head + p.tokens - tail <= 0) return;
  const int64_t per_row = static_cast<int64_t>(p.heads) * (D / 8);
  const int64_t outside = (static_cast<int64_t>(head) + p.tokens - tail) * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + 64 * wave + fresh_lane(); i < outside;
       i += static_cast<int64_t>(n_blocks) * kThreads) {
    const int64_t at = i < head * per_row ? i : i + (static_cast<int64_t>(tail) - head) * per_row;
    const uint4 zero = {0, 0, 0, 0};
    static_cast<uint4 *>(p.out)[at] = zero;
  }
}

// Zeroes the arrival counters of a call whose stream has no counter slot.
__global__ void zero_counters_kernel(unsigned *counters, int n) {
  const int i = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
  if (i < n) counters[i] = 0;
}

int attend_blocks(int head_dim) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  return (head_dim == 64 ? Geo<64>::kBlocks : Geo<128>::kBlocks) * device_cu_count(dev);
}
int slot_rows_of(int tokens, int group) {
  return static_cast<int64_t>(tokens) * group <= kNarrowRows ? kNarrowRows : kWideRows;
}

template <typename T, int D>
int launch(const AttendPagedParams &p, int n_blocks, hipStream_t stream) {
  hipLaunchKernelGGL((attend_paged_kernel<T, D>), dim3(static_cast<unsigned>(n_blocks)),
                     dim3(kThreads), 0, stream, p);
  return check_hip(hipGetLastError(), "attend_paged_kernel launch");
}

size_t counter_bytes(size_t n) { return (n * sizeof(unsigned) + 255) / 256 * 256; }

}  // namespace

size_t attend_paged_workspace_bytes(int tokens, int group, int head_dim) {
  const size_t n = static_cast<size_t>(attend_blocks(head_dim));
  return counter_bytes(n) +
         2 * n * slot_rows_of(tokens, group) * (static_cast<size_t>(head_dim) + 2) * sizeof(float);
}

int launch_attend_paged(AttendPagedParams p, bool bf16, int head_dim, float scale, void *workspace,
                        hipStream_t stream) {
  const int n_blocks = attend_blocks(head_dim);
  if (n_blocks <= 0) return set_error(FA_ERR_HIP, "could not query the compute-unit count");
  p.group = p.heads / p.kv_heads;
  p.slot_rows = slot_rows_of(p.tokens, p.group);
  p.capacity = p.max_pages << p.page_shift;
  p.wide_tokens = kWideRows / p.group;
  p.narrow_tokens = kNarrowRows / p.group;
  p.head_bytes = static_cast<unsigned>((head_dim * 2) << p.page_shift);
  p.page_bytes = p.head_bytes * static_cast<unsigned>(p.kv_heads);
  p.narrow_step = kWaves * kNarrowKeys / kTileKeys;
  p.wide_inv = 1.0f / static_cast<float>(p.wide_tokens);
  p.group_inv = (65536 + p.group - 1) / p.group;
  // Weight of any batch of this many tokens and sequences (those without tokens have none).
  const double tiles = static_cast<double>(p.tokens) / p.wide_tokens + min(p.batch, p.tokens);
  if (tiles * p.kv_heads > 5e8)
    return set_error(FA_ERR_INVALID_ARGUMENT, "too many query tiles: %d tokens, H=%d H_kv=%d",
                     p.tokens, p.heads, p.kv_heads);
  const double most =
      tiles * p.kv_heads * (2.0 + p.capacity + kItemKeys + p.tokens + 2.0 * p.wide_tokens);
  p.unit = 0;
  while (most / static_cast<double>(1u << p.unit) + tiles * p.kv_heads > 1e9 && p.unit < 30) ++p.unit;
  p.blocks_inv = static_cast<unsigned>(0xffffffffu / static_cast<unsigned>(n_blocks));
  p.min_share = (kMinShareKeys >> p.unit) + 1;
  // A negative scale negates q (exactly), so that the row bound is a maximum; a
  // zero one becomes the least that keeps a hidden key's -inf (-inf * 0 is NaN).
  p.negate = scale < 0.f;
  p.c = fmaxf(fabsf(scale) * kLog2e, 1e-37f);
  p.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                         counter_bytes(static_cast<size_t>(n_blocks)));
  // Arrival counters: the stream's own, zero between calls, or, where it has no slot,
  // the workspace's, zeroed by a launch of their own.
  p.counters = merge_counters(kPagedCounters, stream, static_cast<size_t>(n_blocks));
  if (p.counters == nullptr) {
    p.counters = static_cast<unsigned *>(workspace);
    hipLaunchKernelGGL(zero_counters_kernel, dim3(static_cast<unsigned>((n_blocks + 255) / 256)),
                       dim3(256), 0, stream, p.counters, n_blocks);
    const int rc = check_hip(hipGetLastError(), "zero_counters_kernel launch");
    if (rc != FA_OK) return rc;
  }
  if (head_dim == 64)
    return bf16 ? launch<__bf16, 64>(p, n_blocks, stream) : launch<_Float16, 64>(p, n_blocks, stream);
  return bf16 ? launch<__bf16, 128>(p, n_blocks, stream) : launch<_Float16, 128>(p, n_blocks, stream);
}

}  // namespace fa
