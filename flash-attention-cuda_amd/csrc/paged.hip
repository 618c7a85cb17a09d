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
//            query head) pair of the K/V head's group, so K and V are read once
//            for the whole group. A sequence of at most 32 rows is one "narrow"
//            item; others are tiles of up to 128 rows of whole tokens.
//   share  = the items laid end to end, weighted by the keys they see, are cut
//            into equal shares, one per block (two blocks per CU): ragged
//            lengths and few sequences fill the chip alike, without a host
//            that knows the lengths. Each block finds its own share from
//            seq_lens and cu_tokens.
//   merge  = an item that a share's border cuts leaves one fp32 partial (O, m,
//            l) per share in the workspace, and a second launch joins them in
//            the order of the shares, so results do not depend on timing.
//
// Block: 256 threads, 4 waves, two blocks per CU.
//   wide item: wave w owns query rows [32 w, +32); the waves share 64-key K and V
//     tiles in an LDS ring filled by direct global->LDS loads.
//   narrow item: the waves take key tiles in turn, each with K and V tiles of its
//     own in LDS (no barrier in the loop), and join their states at the end.
//   Products on v_mfma_f32_32x32x16: S^T = K Q^T, O^T += V^T P^T (mfma_tile.h), a
//   query row per lane pair.
//
// Roundings to 16 bits. P is rounded once on wide items (the row sum is taken of
// the rounded weights, so a row that one key carries is exact) and split into two
// parts on narrow ones, where memory is what bounds the loop.
//
// Memory safety. Lengths, bounds and page ids are device data, which the host
// cannot check: token ranges are clamped to the packed tensors, key ranges to the
// page table's width, and a page id outside the pool is replaced by page 0 for
// the address and its keys are masked out. V rows past a sequence's end
// are cleared in LDS before they meet a weight of zero (0 * NaN).

#include "mfma_tile.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kTileKeys = 64;     // keys per tile of a wide item, and the unit of a share's border
constexpr int kWideRows = 128;    // query rows of a wide item
constexpr int kNarrowRows = 32;   // most query rows of a narrow item
constexpr int kRingBytes = 64 * 1024;
constexpr int kMergeRows = 8;     // rows per merge block
constexpr int kItemKeys = 128;    // an item's fixed cost, in keys
constexpr int kMinShareKeys = 256;  // least weight of a share
constexpr int kSnapTiles = 1;     // borders this close to an item's end move there

template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef half8 type;
  typedef half2 pair;
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
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
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

// ---- sequences, items and shares ------------------------------------------------

// A sequence's new tokens: packed rows [t0, t0 + n), the first at position p0.
struct Seq {
  int t0, n, p0;
};
__device__ __forceinline__ Seq load_seq(const AttendPagedParams &p, int b) {
  const int lo = p.cu_tokens[b], hi = p.cu_tokens[b + 1];
  Seq s;
  s.t0 = min(max(lo, 0), p.tokens);
  s.n = min(max(hi, s.t0), p.tokens) - s.t0;
  // seq_lens - hi + t0, kept far from overflow whatever the buffers hold.
  const int64_t p0 = static_cast<int64_t>(p.seq_lens[b]) - hi + s.t0;
  s.p0 = static_cast<int>(min(max(p0, static_cast<int64_t>(-(1 << 30))),
                              static_cast<int64_t>(1 << 30)));
  return s;
}
// Items of a sequence (per K/V head): `count` tiles of `tokens` tokens.
struct Tiles {
  int count, tokens;
};
__device__ __forceinline__ Tiles tiles_of(const AttendPagedParams &p, int n) {
  Tiles t;
  const bool narrow = n <= kNarrowRows / p.group;
  t.tokens = narrow ? max(n, 1) : kWideRows / p.group;
  t.count = narrow ? (n > 0 ? 1 : 0) : (n + t.tokens - 1) / t.tokens;
  return t;
}
// Keys the last token of a tile sees.
__device__ __forceinline__ int key_end(const AttendPagedParams &p, const Seq &s, const Tiles &t,
                                       int tile) {
  const int64_t last = static_cast<int64_t>(s.p0) +
                       min(static_cast<int64_t>(s.n), static_cast<int64_t>(tile + 1) * t.tokens);
  return static_cast<int>(min(max(last, int64_t{0}), static_cast<int64_t>(p.capacity)));
}
// Weight of tiles [0, tile) of one K/V head: the keys each tile sees (taken as
// if the last tile were whole) plus a fixed cost per item.
__device__ __forceinline__ int64_t weight_before(const AttendPagedParams &p, const Seq &s,
                                                 const Tiles &t, int tile) {
  const int64_t each = static_cast<int64_t>(min(max(s.p0, 0), p.capacity)) + kItemKeys;
  return tile * each + static_cast<int64_t>(t.tokens) * tile * (tile + 1) / 2;
}

// A share's border: before key tile `kt` of item (b, kvh, tile).
struct Border {
  int b, kvh, tile, kt;
};
__device__ __forceinline__ bool same_item(const Border &a, const Border &b) {
  return a.b == b.b && a.kvh == b.kvh && a.tile == b.tile;
}

// The border at weight `at` inside sequence b (0 <= at < H_kv * whole).
__device__ Border border_in(const AttendPagedParams &p, const Seq &s, const Tiles &t, int b,
                            int64_t whole, int64_t at) {
  Border r;
  r.b = b;
  r.kvh = static_cast<int>(at / whole);
  at -= r.kvh * whole;
  int lo = 0, hi = t.count;  // the last tile whose weight_before is <= at
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (weight_before(p, s, t, mid) <= at) lo = mid;
    else hi = mid;
  }
  r.tile = lo;
  const int tiles = (key_end(p, s, t, lo) + kTileKeys - 1) / kTileKeys;
  const int64_t in = at - weight_before(p, s, t, lo) - kItemKeys;
  r.kt = static_cast<int>(min(max(in, int64_t{0}) / kTileKeys, static_cast<int64_t>(tiles)));
  // A border close to an item's end moves there: a partial costs more than the keys it balances.
  if (r.kt < kSnapTiles) r.kt = 0;
  else if (r.kt > tiles - kSnapTiles) r.kt = tiles;
  return r;
}

// Record of a share's first border, kept for the merge launch.
struct Record {
  Border at;
  int tiles;   // key tiles of that item
  int t0, n;   // its packed tokens
  int pad;
};
static_assert(sizeof(Record) == 32, "two 16-byte pieces");

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

// Loads the lane's query row `row` of an item (rows past the last repeat it).
template <typename T, int D>
__device__ __forceinline__ void load_queries(const AttendPagedParams &p, int t0, int n, int p0,
                                             int kvh, int row, int g, Rows<T, D> &r) {
  row = min(row, n * p.group - 1);
  const int token = row / p.group;
  const int head = kvh * p.group + row - token * p.group;
  const T *q = static_cast<const T *>(p.q) + static_cast<int64_t>(t0 + token) * p.q_token +
               static_cast<int64_t>(head) * p.q_head;
  r.pos = p0 + token;
  const unsigned flip = p.negate ? 0x80008000u : 0u;  // a negative scale: -q, exactly
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    uint4 x = *reinterpret_cast<const uint4 *>(q + (D / 2) * g + 8 * s);
    x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
    r.q[s] = __builtin_bit_cast(frag_t<T>, x);
  }
}

// ---- one tile of KB 32-key blocks: scores, softmax, products ------------------------

// Scores of the tile at LDS byte address `tile`.
template <typename T, int D, int KB>
__device__ __forceinline__ void scores(unsigned tile, const FragOffsetsD<D> &fo,
                                       const Rows<T, D> &r, floatx16 (&s)[KB]) {
  typedef __attribute__((address_space(3))) const frag_t<T> lds_frag;
  const unsigned base = uniform_lds_u(tile);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a) s[kb][a] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    lds_half *at = opaque_lds_at(base, fo.k[i]);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const frag_t<T> k = *reinterpret_cast<lds_frag *>(at + kb * 32 * D);
      s[kb] = Frag<T>::mm(k, r.q[i], s[kb]);
    }
  }
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

// Weights of the tile as P^T fragments (SPLIT: lo holds what hi lost). The bound m
// moves only when a row's scores pass it by more than 2^8 (weights up to 2^8 are
// harmless in either type): O is rescaled a few times per item instead of per tile.
template <typename T, int D, int KB, bool SPLIT>
__device__ __forceinline__ void weigh(floatx16 (&s)[KB], float c, Rows<T, D> &r,
                                      frag_t<T> (&hi)[2 * KB], frag_t<T> (&lo)[2 * KB]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int a = 0; a < 16; ++a) mx = fmaxf(mx, s[kb][a]);
  mx = max_lane_pair(mx) * c;
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
    for (int a = 0; a < 16; ++a) {
      const float w = fast_exp2(__builtin_fmaf(s[kb][a], c, -m));
      const T h = static_cast<T>(w);
      hi[2 * kb + (a >> 3)][a & 7] = h;
      if constexpr (SPLIT) lo[2 * kb + (a >> 3)][a & 7] = static_cast<T>(w - static_cast<float>(h));
    }
}

template <typename T, int D, int KB, bool SPLIT>
__device__ __forceinline__ void accumulate(unsigned tile, const FragOffsetsD<D> &fo,
                                           const frag_t<T> &ones, const frag_t<T> (&hi)[2 * KB],
                                           const frag_t<T> (&lo)[2 * KB], Rows<T, D> &r) {
  const unsigned base = uniform_lds_u(tile);
#pragma unroll
  for (int ks = 0; ks < 2 * KB; ++ks) {
    r.l = Frag<T>::mm16(ones, hi[ks], r.l);
    if constexpr (SPLIT) r.l = Frag<T>::mm16(ones, lo[ks], r.l);
  }
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
    lds_half *at = opaque_lds_at(base, fo.v[db]);
#pragma unroll
    for (int ks = 0; ks < 2 * KB; ++ks) {
      frag_t<T> v;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4v *)(at + (ks * 16 + 8 * part) * D));
        typedef T t4 __attribute__((ext_vector_type(4)));
        const t4 y = __builtin_bit_cast(t4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * part + e] = y[e];
      }
      r.o[db] = Frag<T>::mm(v, hi[ks], r.o[db]);
      if constexpr (SPLIT) r.o[db] = Frag<T>::mm(v, lo[ks], r.o[db]);
    }
  }
}

// ---- pages --------------------------------------------------------------------------

typedef const __attribute__((address_space(4))) int32_t *uniform_table;

// Where 16 consecutive keys of one K/V head begin; `absent` where their page id
// is outside the pool (the address is page 0's then).
struct Slab {
  int64_t at;  // in rows of head_dim elements
  bool absent;
};
__device__ __forceinline__ Slab slab_of(const AttendPagedParams &p, uniform_table table, int kvh,
                                        int key, int end) {
  // Keys past the end lie on no page of their own: the last key's page stands in.
  if (key >= end) key = (end - 1) & ~15;
  const int page = __builtin_amdgcn_readfirstlane(table[key >> p.page_shift]);
  Slab s;
  s.absent = static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages);
  const int64_t id = s.absent ? 0 : page;
  s.at = ((id * p.kv_heads + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
  return s;
}

// Per-lane source offsets (bytes) of the 16-byte pieces that fill 16 rows of a K
// or V tile; a load instruction writes 1 KiB of LDS, 64 / (D / 8) rows.
template <int D>
struct LoadOffsets {
  static constexpr int kLoads = D / 32;  // instructions per 16 rows
  unsigned k[kLoads], v[kLoads];
};
template <int D>
__device__ __forceinline__ LoadOffsets<D> load_offsets(int lane) {
  LoadOffsets<D> lo;
  constexpr int kChunks = D / 8;
#pragma unroll
  for (int j = 0; j < LoadOffsets<D>::kLoads; ++j) {
    const int row = j * (64 / kChunks) + lane / kChunks;
    const int chunk = lane % kChunks;
    lo.k[j] = static_cast<unsigned>(row * D + ((chunk ^ k_swz_d<D>(row)) << 3)) * 2;
    lo.v[j] = static_cast<unsigned>(row * D + ((chunk ^ v_swz_d<D>(row)) << 3)) * 2;
  }
  return lo;
}
template <int D>
__device__ __forceinline__ void load_slab(const void *pages, int64_t at,
                                          const unsigned (&off)[LoadOffsets<D>::kLoads],
                                          unsigned lds, bool once) {
  const char *base = static_cast<const char *>(pages) + at * (D * 2);
#pragma unroll
  for (int j = 0; j < LoadOffsets<D>::kLoads; ++j) {
    if (once) global_to_lds16_sbase_nt_at(base, off[j], lds + 1024 * j);
    else global_to_lds16_sbase_at(base, off[j], lds + 1024 * j);
  }
}

// ---- results -------------------------------------------------------------------------

// Partial of a share: rows of D floats, then (m, l) pairs.
__device__ __forceinline__ float *partial_of(const AttendPagedParams &p, int slot, int head_dim) {
  return p.partials + static_cast<int64_t>(slot) * p.slot_rows * (head_dim + 2);
}

template <typename T>
__device__ __forceinline__ T *out_row(const AttendPagedParams &p, int t0, int kvh, int row,
                                      int head_dim) {
  const int token = row / p.group;
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

struct Item {
  int t0, n, p0;     // packed tokens and the first one's position
  int kvh;
  int kt0, kt1;      // key tiles of this share
  int end;           // keys the item sees (the last token's)
  int slot;          // partial slot, -1: the whole item
  uniform_table table;
};

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

template <typename T, int D>
__device__ __forceinline__ void wide_item(const AttendPagedParams &p, const Item &it,
                                          unsigned ring) {
  constexpr int kTileBytes = kTileKeys * D * 2;
  constexpr int kStages = kRingBytes / (2 * kTileBytes);
  constexpr int kLoads = 2 * LoadOffsets<D>::kLoads;  // a wave's loads per tile
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  const int rows = it.n * p.group;
  const int row = 32 * wave + (lane & 31);
  const FragOffsetsD<D> fo = frag_offsets_d<D>(lane);
  const LoadOffsets<D> lo = load_offsets<D>(lane);
  const frag_t<T> ones = ones_selector<T>(lane);
  Rows<T, D> r;
  load_queries<T, D>(p, it.t0, it.n, it.p0, it.kvh, row, g, r);
  clear_rows<T, D>(r);
  // Positions of the wave's first and last query.
  const int first_pos = it.p0 + min(32 * wave, rows - 1) / p.group;
  const int last_pos = it.p0 + min(32 * wave + 31, rows - 1) / p.group;
  const bool has_rows = 32 * wave < rows;

  // Wave w loads rows [16 w, +16) of each tile's K and V.
  auto issue = [&](int kt) {
    const int stage = (kt - it.kt0) % kStages;
    const Slab s = slab_of(p, it.table, it.kvh, kt * kTileKeys + 16 * wave, it.end);
    const unsigned at = ring + stage * 2 * kTileBytes + 16 * wave * D * 2;
    load_slab<D>(p.k_pages, s.at, lo.k, at, false);
    load_slab<D>(p.v_pages, s.at, lo.v, at + kTileBytes, false);
  };
  auto absent_rows = [&](int kt) {
    unsigned absent = 0;
#pragma unroll
    for (int i = 0; i < kTileKeys / 16; ++i)
      absent |= slab_of(p, it.table, it.kvh, kt * kTileKeys + 16 * i, it.end).absent ? 1u << i : 0u;
    return absent;
  };

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i)
    if (it.kt0 + i < it.kt1) issue(it.kt0 + i);
  for (int kt = it.kt0; kt < it.kt1; ++kt) {
    // Tile kt has landed once at most the later tiles' loads are outstanding.
    const int later = min(kStages - 2, it.kt1 - 1 - kt);
    if (kStages > 2 && later >= 2) wait_loads<2 * kLoads>();
    else if (kStages > 2 && later == 1) wait_loads<kLoads>();
    else wait_loads<0>();
    block_barrier();
    if (kt + kStages - 1 < it.kt1) issue(kt + kStages - 1);
    const unsigned k_tile = ring + ((kt - it.kt0) % kStages) * 2 * kTileBytes;
    const unsigned v_tile = k_tile + kTileBytes;
    const int key0 = kt * kTileKeys;
    const unsigned absent = absent_rows(kt);
    if (absent != 0 || key0 + kTileKeys > it.end) {
      clear_v<D>(v_tile, kTileKeys, it.end - key0, absent, threadIdx.x, kThreads);
      block_barrier();
    }
    if (!has_rows || last_pos < key0) continue;
    floatx16 s[2];
    frag_t<T> hi[4], none[4];
    scores<T, D, 2>(k_tile, fo, r, s);
    if (absent != 0 || first_pos < key0 + kTileKeys - 1 || key0 + kTileKeys > it.end)
      hide<2>(s, min(r.pos, it.end - 1) - key0 - 4 * g, absent);
    weigh<T, D, 2, false>(s, p.c, r, hi, none);
    accumulate<T, D, 2, false>(v_tile, fo, ones, hi, none, r);
  }
  block_barrier();  // the ring may be filled for the next item

  if (row >= rows) return;
  const float l = r.l[0];
  if (it.slot < 0) {
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;  // NaN stays NaN
    T *o = out_row<T>(p, it.t0, it.kvh, row, D);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx4 x = {r.o[i][4 * a] * inv, r.o[i][4 * a + 1] * inv, r.o[i][4 * a + 2] * inv,
                           r.o[i][4 * a + 3] * inv};
        store4<T>(o + 32 * i + 8 * a + 4 * g, x);
      }
  } else {
    float *part = partial_of(p, it.slot, D);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx4 x = {r.o[i][4 * a], r.o[i][4 * a + 1], r.o[i][4 * a + 2], r.o[i][4 * a + 3]};
        *reinterpret_cast<floatx4 *>(part + row * D + 32 * i + 8 * a + 4 * g) = x;
      }
    if (g == 0) {
      float *ml = part + p.slot_rows * D + 2 * row;
      ml[0] = r.m;
      ml[1] = l;
    }
  }
}

template <typename T, int D>
__device__ __forceinline__ void narrow_item(const AttendPagedParams &p, const Item &it,
                                            unsigned ring, float *exchange, float *exchange_ml) {
  constexpr int kKeys = 4096 / D;  // keys of a wave's 8 KiB tile
  constexpr int KB = kKeys / 32;
  constexpr int kTileBytes = 8192;
  constexpr int kLoads = 8;        // load instructions per tile
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5;
  const int rows = it.n * p.group;
  const FragOffsetsD<D> fo = frag_offsets_d<D>(lane);
  const LoadOffsets<D> lo = load_offsets<D>(lane);
  const frag_t<T> ones = ones_selector<T>(lane);
  const unsigned k_tile = ring + wave * 2 * kTileBytes, v_tile = k_tile + kTileBytes;
  const int stop = min(it.end, it.kt1 * kTileKeys);
  auto issue = [&](const void *pages, const unsigned (&off)[LoadOffsets<D>::kLoads], unsigned lds,
                   int key0) {
    unsigned absent = 0;
#pragma unroll
    for (int i = 0; i < kKeys / 16; ++i) {
      const Slab s = slab_of(p, it.table, it.kvh, key0 + 16 * i, it.end);
      absent |= s.absent ? 1u << i : 0u;
      load_slab<D>(pages, s.at, off, lds + 16 * i * D * 2, true);
    }
    return absent;
  };
  int key0 = it.kt0 * kTileKeys + wave * kKeys;
  unsigned absent = 0;
  if (key0 < stop) {
    absent = issue(p.k_pages, lo.k, k_tile, key0);
    issue(p.v_pages, lo.v, v_tile, key0);
  }
  Rows<T, D> r;
  load_queries<T, D>(p, it.t0, it.n, it.p0, it.kvh, lane & 31, g, r);
  clear_rows<T, D>(r);
  for (; key0 < stop; key0 += kWaves * kKeys) {
    const int next = key0 + kWaves * kKeys;
    // Loads leave in the order K, V, K, V: at most the 8 of V are younger than K's.
    wait_loads<kLoads>();
    floatx16 s[KB];
    frag_t<T> hi[2 * KB], low[2 * KB];
    scores<T, D, KB>(k_tile, fo, r, s);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read before it is overwritten
    unsigned next_absent = 0;
    if (next < stop) next_absent = issue(p.k_pages, lo.k, k_tile, next);
    if (absent != 0 || it.p0 < key0 + kKeys - 1 || key0 + kKeys > it.end)
      hide<KB>(s, min(r.pos, it.end - 1) - key0 - 4 * g, absent);
    weigh<T, D, KB, true>(s, p.c, r, hi, low);
    if (next < stop) wait_loads<kLoads>();
    else wait_loads<0>();
    if (absent != 0 || key0 + kKeys > it.end) {
      clear_v<D>(v_tile, kKeys, it.end - key0, absent, lane, kWave);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    accumulate<T, D, KB, true>(v_tile, fo, ones, hi, low, r);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next < stop) issue(p.v_pages, lo.v, v_tile, next);
    absent = next_absent;
  }

  // Join the four waves' states. Row r's dims lie in LDS as 16-byte pieces,
  // piece j at j ^ (r & 15).
  block_barrier();  // every wave is done with its tiles
  const int row = lane & 31;
  if (row < rows) {
    float *x = exchange + (wave * kNarrowRows + row) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx4 o = {r.o[i][4 * a], r.o[i][4 * a + 1], r.o[i][4 * a + 2], r.o[i][4 * a + 3]};
        *reinterpret_cast<floatx4 *>(x + 4 * ((8 * i + 2 * a + g) ^ (row & 15))) = o;
      }
    if (g == 0) {
      exchange_ml[2 * (wave * kNarrowRows + row)] = r.m;
      exchange_ml[2 * (wave * kNarrowRows + row) + 1] = r.l[0];
    }
  }
  block_barrier();
  for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
    const int at = i / (D / 4), piece = i % (D / 4);
    float m = -INFINITY, l = 0.f;
    float w[kWaves];
#pragma unroll
    for (int j = 0; j < kWaves; ++j) m = fmaxf(m, exchange_ml[2 * (j * kNarrowRows + at)]);
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      const float mj = exchange_ml[2 * (j * kNarrowRows + at)];
      w[j] = mj == -INFINITY ? 0.f : fast_exp2(mj - m);
      l += w[j] * exchange_ml[2 * (j * kNarrowRows + at) + 1];
      const floatx4 x = *reinterpret_cast<const floatx4 *>(
          exchange + (j * kNarrowRows + at) * D + 4 * (piece ^ (at & 15)));
      if (mj != -INFINITY) o += w[j] * x;
    }
    if (it.slot < 0) {
      const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
      o *= inv;
      store4<T>(out_row<T>(p, it.t0, it.kvh, at, D) + 4 * piece, o);
    } else {
      float *part = partial_of(p, it.slot, D);
      *reinterpret_cast<floatx4 *>(part + at * D + 4 * piece) = o;
      if (piece == 0) {
        part[p.slot_rows * D + 2 * at] = m;
        part[p.slot_rows * D + 2 * at + 1] = l;
      }
    }
  }
  block_barrier();  // the exchange may be overwritten
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_paged_kernel(const AttendPagedParams p) {
  __shared__ __align__(1024) unsigned char ring_mem[kRingBytes];
  __shared__ __align__(16) float ml_mem[2 * kWaves * kNarrowRows];
  __shared__ int64_t wave_weight[kWaves];
  __shared__ Border borders[2];

  Record *records = static_cast<Record *>(p.records);
  const int tid = static_cast<int>(threadIdx.x);
  const int n_blocks = static_cast<int>(gridDim.x);

  // Outputs of packed rows that belong to no sequence are zero.
  {
    const int lo = min(max(p.cu_tokens[0], 0), p.tokens);
    const int hi = min(max(p.cu_tokens[p.batch], 0), p.tokens);
    const int64_t per_row = static_cast<int64_t>(p.heads) * (D / 8);
    const int64_t outside = (static_cast<int64_t>(lo) + p.tokens - hi) * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < outside;
         i += static_cast<int64_t>(n_blocks) * kThreads) {
      const int64_t at = i < lo * per_row ? i : i + (static_cast<int64_t>(hi) - lo) * per_row;
      const uint4 zero = {0, 0, 0, 0};
      static_cast<uint4 *>(p.out)[at] = zero;
    }
  }

  // Every block sums the sequences' weights and finds its share's two borders.
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = load_seq(p, b);
    const Tiles t = tiles_of(p, s.n);
    mine += weight_before(p, s, t, t.count) * p.kv_heads;
  }
  int64_t before = mine;  // inclusive sum over the wave
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t x = __shfl_up(before, d);
    if ((tid & 63) >= d) before += x;
  }
  if ((tid & 63) == 63) wave_weight[tid >> 6] = before;
  if (tid < 2) borders[tid] = Border{p.batch, 0, 0, 0};
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < (tid >> 6)) before += wave_weight[w];
    total += wave_weight[w];
  }
  before -= mine;
  const int64_t share =
      max((total + n_blocks - 1) / n_blocks, static_cast<int64_t>(kMinShareKeys));
  const int active = static_cast<int>((total + share - 1) / share);
  // Neighbouring shares read the same keys, so they go to one XCD (blocks are
  // dealt to the 8 XCDs in turn).
  const int per_xcd = (active + 7) / 8;
  const int blk = static_cast<int>(blockIdx.x);
  const int w = blk < 8 * per_xcd ? (blk & 7) * per_xcd + (blk >> 3) : blk;
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int64_t at = (w + side) * share;
    if (at < before || at >= before + mine) continue;
    int64_t from = before;
    for (int b = b0; b < b1; ++b) {
      const Seq s = load_seq(p, b);
      const Tiles t = tiles_of(p, s.n);
      const int64_t whole = weight_before(p, s, t, t.count);
      if (at < from + whole * p.kv_heads) {
        borders[side] = border_in(p, s, t, b, whole, at - from);
        break;
      }
      from += whole * p.kv_heads;
    }
  }
  __syncthreads();
  Border cur = borders[0], end = borders[1];
  cur.b = __builtin_amdgcn_readfirstlane(cur.b);
  cur.kvh = __builtin_amdgcn_readfirstlane(cur.kvh);
  cur.tile = __builtin_amdgcn_readfirstlane(cur.tile);
  cur.kt = __builtin_amdgcn_readfirstlane(cur.kt);
  end.b = __builtin_amdgcn_readfirstlane(end.b);
  end.kvh = __builtin_amdgcn_readfirstlane(end.kvh);
  end.tile = __builtin_amdgcn_readfirstlane(end.tile);
  end.kt = __builtin_amdgcn_readfirstlane(end.kt);

  const unsigned ring = lds_addr(ring_mem);
  bool first = true;
  Seq s = {0, 0, 0};
  Tiles t = {0, 1};
  int loaded = -1;
  for (;;) {
    if (cur.b >= p.batch) break;
    if (loaded != cur.b) {
      s = load_seq(p, cur.b);
      s.t0 = __builtin_amdgcn_readfirstlane(s.t0);
      s.n = __builtin_amdgcn_readfirstlane(s.n);
      s.p0 = __builtin_amdgcn_readfirstlane(s.p0);
      t = tiles_of(p, s.n);
      loaded = cur.b;
    }
    if (cur.tile >= t.count) {  // next K/V head or sequence
      cur.tile = 0;
      cur.kt = 0;
      if (t.count == 0 || ++cur.kvh >= p.kv_heads) {
        cur.kvh = 0;
        ++cur.b;
      }
      if (cur.b > end.b) break;
      continue;
    }
    const bool last = same_item(cur, end);
    Item it;
    it.end = key_end(p, s, t, cur.tile);
    const int tiles = (it.end + kTileKeys - 1) / kTileKeys;
    it.kt0 = cur.kt;
    it.kt1 = last ? min(end.kt, tiles) : tiles;
    it.t0 = s.t0 + cur.tile * t.tokens;
    it.n = min(t.tokens, s.n - cur.tile * t.tokens);
    it.p0 = s.p0 + cur.tile * t.tokens;
    it.kvh = cur.kvh;
    it.table = (uniform_table)(reinterpret_cast<uintptr_t>(
        p.page_table + static_cast<int64_t>(cur.b) * p.max_pages));
    if (first && tid == 0) {
      Record rec;
      rec.at = cur;
      rec.tiles = tiles;
      rec.t0 = it.t0;
      rec.n = it.n;
      rec.pad = 0;
      records[w] = rec;
    }
    first = false;
    // A whole item (also one that sees no key) is written out; a part leaves a partial.
    const bool whole = it.kt0 == 0 && it.kt1 == tiles && !(last && end.kt < tiles) &&
                       !(last && tiles == 0);
    if (whole || it.kt1 > it.kt0) {
      it.slot = whole ? -1 : 2 * w + (it.kt0 == 0 ? 1 : 0);
      if (it.n * p.group <= kNarrowRows)
        narrow_item<T, D>(p, it, ring, reinterpret_cast<float *>(ring_mem), ml_mem);
      else
        wide_item<T, D>(p, it, ring);
    }
    if (last) break;
    ++cur.tile;
    cur.kt = 0;
  }
  if (first && tid == 0) {
    Record rec;
    rec.at = Border{-1, 0, 0, 0};
    rec.tiles = rec.t0 = rec.n = rec.pad = 0;
    records[w] = rec;
  }
}

// Joins the partials of an item that borders cut: block (w, y) takes rows
// [8 y, +8) of the item whose first inner border is share w's.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attend_merge_kernel(const AttendPagedParams p,
                                                                int n_blocks) {
  const Record *records = static_cast<const Record *>(p.records);
  const int w = static_cast<int>(blockIdx.x) + 1;
  const Record rec = records[w];
  if (rec.at.b < 0 || rec.at.kt <= 0) return;
  const Record prev = records[w - 1];
  if (same_item(prev.at, rec.at) && prev.at.kt > 0) return;
  if (rec.at.kt >= rec.tiles) return;  // the share before holds the whole item
  const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
  constexpr int kPer = D / 64;  // dims per lane
  for (int row = kMergeRows * blockIdx.y + wave; row < kMergeRows * (static_cast<int>(blockIdx.y) + 1);
       row += kWaves) {
    if (row >= rec.n * p.group) return;
    float m = -INFINITY, l = 0.f, o[kPer] = {};
    auto add = [&](int slot) {
      const float *part = partial_of(p, slot, D);
      const float pm = part[p.slot_rows * D + 2 * row];
      const float pl = part[p.slot_rows * D + 2 * row + 1];
      float x[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = part[row * D + kPer * lane + i];
      if (pm == -INFINITY) return;
      const float top = fmaxf(m, pm);
      const float a = m == -INFINITY ? 0.f : fast_exp2(m - top), b = fast_exp2(pm - top);
      m = top;
      l = l * a + pl * b;
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] = o[i] * a + x[i] * b;
    };
    add(2 * (w - 1) + 1);
    int kt = rec.at.kt;
    for (int j = w; j < n_blocks && kt < rec.tiles; ++j) {
      int next = rec.tiles;
      if (j + 1 < n_blocks) {
        const Record r = records[j + 1];
        if (r.at.b >= 0 && same_item(r.at, rec.at)) next = r.at.kt;
      }
      if (next > kt) add(2 * j);
      kt = next;
    }
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
    T *out = out_row<T>(p, rec.t0, rec.at.kvh, row, D) + kPer * lane;
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] = static_cast<T>(o[i] * inv);
  }
}

int attend_blocks() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  return 2 * device_cu_count(dev);
}
int slot_rows_of(int tokens, int group) {
  return static_cast<int>(
      min(static_cast<int64_t>(kWideRows), static_cast<int64_t>(tokens) * group));
}

template <typename T, int D>
int launch(const AttendPagedParams &p, int n_blocks, hipStream_t stream) {
  hipLaunchKernelGGL((attend_paged_kernel<T, D>), dim3(static_cast<unsigned>(n_blocks)),
                     dim3(kThreads), 0, stream, p);
  int rc = check_hip(hipGetLastError(), "attend_paged_kernel launch");
  if (rc != FA_OK) return rc;
  const unsigned groups = static_cast<unsigned>((p.slot_rows + kMergeRows - 1) / kMergeRows);
  hipLaunchKernelGGL((attend_merge_kernel<T, D>), dim3(static_cast<unsigned>(n_blocks - 1), groups),
                     dim3(kThreads), 0, stream, p, n_blocks);
  return check_hip(hipGetLastError(), "attend_merge_kernel launch");
}

}  // namespace

size_t attend_paged_workspace_bytes(int tokens, int group, int head_dim) {
  const size_t n = static_cast<size_t>(attend_blocks());
  return n * sizeof(Record) +
         2 * n * slot_rows_of(tokens, group) * (static_cast<size_t>(head_dim) + 2) * sizeof(float);
}

int launch_attend_paged(AttendPagedParams p, bool bf16, int head_dim, float scale, void *workspace,
                        hipStream_t stream) {
  const int n_blocks = attend_blocks();
  if (n_blocks <= 0) return set_error(FA_ERR_HIP, "could not query the compute-unit count");
  p.group = p.heads / p.kv_heads;
  p.slot_rows = slot_rows_of(p.tokens, p.group);
  p.capacity = p.max_pages << p.page_shift;
  // A negative scale negates q (exactly), so that the row bound is a maximum; a
  // zero one becomes the least that keeps a hidden key's -inf (-inf * 0 is NaN).
  p.negate = scale < 0.f;
  p.c = fmaxf(fabsf(scale) * kLog2e, 1e-37f);
  p.records = workspace;
  p.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                         static_cast<size_t>(n_blocks) * sizeof(Record));
  if (head_dim == 64)
    return bf16 ? launch<__bf16, 64>(p, n_blocks, stream) : launch<_Float16, 64>(p, n_blocks, stream);
  return bf16 ? launch<__bf16, 128>(p, n_blocks, stream) : launch<_Float16, 128>(p, n_blocks, stream);
}

}  // namespace fa
