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
//            l) per share in the workspace; the block that finishes last joins
//            them in the order of the shares, so results do not depend on timing.
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

// Key tiles of an item.
__device__ __forceinline__ int key_tiles(int end) { return (end + kTileKeys - 1) / kTileKeys; }

// floor(a / b) for 0 <= a < 2^52, b > 0: a product in fp64 (one estimate off by at
// most one, then corrected) instead of a 64-bit integer division, which costs
// over a hundred dependent instructions at the start of every block.
__device__ __forceinline__ int64_t floor_div(int64_t a, int64_t b) {
  int64_t q = static_cast<int64_t>(static_cast<double>(a) / static_cast<double>(b));
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}
__device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return floor_div(a + b - 1, b); }

// A share's border: before key tile `kt` of item (b, kvh, tile); `from` is the weight
// of the sequences before b.
struct Border {
  int b, kvh, tile, kt;
  Seq s;
  int pad;
  int64_t from;
};

// The border at weight `at` inside sequence b (0 <= at - from < H_kv * whole).
__device__ Border border_in(const AttendPagedParams &p, const Seq &s, const Tiles &t, int b,
                            int64_t whole, int64_t from, int64_t at) {
  Border r;
  r.b = b;
  r.s = s;
  r.from = from;
  at -= from;
  r.kvh = static_cast<int>(floor_div(at, whole));
  at -= r.kvh * whole;
  int lo = 0, hi = t.count;  // the last tile whose weight_before is <= at
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (weight_before(p, s, t, mid) <= at) lo = mid;
    else hi = mid;
  }
  r.tile = lo;
  const int tiles = key_tiles(key_end(p, s, t, lo));
  const int64_t in = at - weight_before(p, s, t, lo) - kItemKeys;
  r.kt = static_cast<int>(min(max(in, int64_t{0}) / kTileKeys, static_cast<int64_t>(tiles)));
  // A border close to an item's end moves there: a partial costs more than the keys it balances.
  if (r.kt < kSnapTiles) r.kt = 0;
  else if (r.kt > tiles - kSnapTiles) r.kt = tiles;
  return r;
}

// The shares that an item of `tiles` key tiles at weights [x0, x1) is cut into: the
// first border inside it and the number of pieces. Piece i is share
// first + i - 1's; a border k lies inside when border_in gives it 0 < kt < tiles.
struct Pieces {
  int first, count;
};
__device__ __forceinline__ Pieces pieces_of(int64_t x0, int64_t x1, int tiles, int64_t share) {
  Pieces r;
  r.first = static_cast<int>(ceil_div(x0 + kItemKeys + kSnapTiles * kTileKeys, share));
  const int64_t stop =
      min(x1, x0 + kItemKeys + static_cast<int64_t>(tiles - kSnapTiles + 1) * kTileKeys);
  r.count = static_cast<int>(ceil_div(stop, share)) - r.first + 1;
  return r;
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

// Partial of a share. Narrow items: rows of D floats, then (m, l) pairs from slot_rows D
// on. Wide items: each wave's accumulators as (pair of elements, lane), then the pairs.
__device__ __forceinline__ float *partial_of(const AttendPagedParams &p, int slot, int head_dim) {
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

// Normalises and stores the lane's half of its query row.
template <typename T, int D>
__device__ __forceinline__ void write_rows(const AttendPagedParams &p, const Item &it, int row,
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

  if (!has_rows) return;
  if (it.slot < 0) {
    write_rows<T, D>(p, it, row, g, r.o, r.l[0]);
  } else {
    float *part = partial_of(p, it.slot, D) + wave * (32 * D) + 2 * lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int a = 0; a < 8; ++a)
        publish2(part + (8 * i + a) * 128, r.o[i][2 * a], r.o[i][2 * a + 1]);
    if (g == 0)
      publish2(partial_of(p, it.slot, D) + kWideRows * D + 2 * row, r.m, r.l[0]);
  }
}

// Joins a wide item's pieces, first to last, and writes its rows.
template <typename T, int D>
__device__ __forceinline__ void join_wide(const AttendPagedParams &p, const Item &it,
                                          const Pieces &pc) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = 32 * wave + (lane & 31);
  if (32 * wave >= it.n * p.group) return;
  float m = -INFINITY, l = 0.f;
  floatx16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int a = 0; a < 16; ++a) o[i][a] = 0.f;
  for (int j = 0; j < pc.count; ++j) {
    const float *part = partial_of(p, 2 * (pc.first + j - 1) + (j == 0 ? 1 : 0), D);
    const floatx2 ml = fetch2(part + kWideRows * D + 2 * row);
    floatx2 x[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; ++i) x[i] = fetch2(part + wave * (32 * D) + 128 * i + 2 * lane);
    const float top = fmaxf(m, ml[0]);
    const float a = m == -INFINITY ? 0.f : fast_exp2(m - top);
    const float b = ml[0] == -INFINITY ? 0.f : fast_exp2(ml[0] - top);
    m = top;
    l = l * a + ml[1] * b;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      o[i / 8][2 * (i % 8)] = o[i / 8][2 * (i % 8)] * a + x[i][0] * b;
      o[i / 8][2 * (i % 8) + 1] = o[i / 8][2 * (i % 8) + 1] * a + x[i][1] * b;
    }
  }
  write_rows<T, D>(p, it, row, lane >> 5, o, l);
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
  for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
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

// Joins a narrow item's pieces, first to last, and writes its rows. Eight pieces' loads are
// in flight at a time.
template <typename T, int D>
__device__ __forceinline__ void join_narrow(const AttendPagedParams &p, const Item &it,
                                            const Pieces &pc) {
  constexpr int kDeep = 8;
  typedef T t2 __attribute__((ext_vector_type(2)));
  const int n = it.n * p.group * (D / 2);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int row = i / (D / 2), at = 2 * (i % (D / 2));
    float m = -INFINITY, l = 0.f;
    floatx2 o = {0.f, 0.f};
    for (int j0 = 0; j0 < pc.count; j0 += kDeep) {
      floatx2 ml[kDeep], x[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int piece = min(j0 + j, pc.count - 1);
        const int share = pc.first + piece - 1;
        const float *part = partial_of(p, 2 * share + (piece == 0 ? 1 : 0), D);
        ml[j] = fetch2(part + p.slot_rows * D + 2 * row);
        x[j] = fetch2(part + row * D + at);
      }
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        if (j0 + j >= pc.count || ml[j][0] == -INFINITY) continue;
        const float top = fmaxf(m, ml[j][0]);
        const float a = m == -INFINITY ? 0.f : fast_exp2(m - top), b = fast_exp2(ml[j][0] - top);
        m = top;
        l = l * a + ml[j][1] * b;
        o = o * a + x[j] * b;
      }
    }
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
    const t2 y = {static_cast<T>(o[0] * inv), static_cast<T>(o[1] * inv)};
    *reinterpret_cast<t2 *>(out_row<T>(p, it.t0, it.kvh, row, D) + at) = y;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_paged_kernel(const AttendPagedParams p) {
  __shared__ __align__(1024) unsigned char ring_mem[kRingBytes];
  __shared__ __align__(16) float ml_mem[2 * kWaves * kNarrowRows];
  __shared__ int64_t wave_weight[kWaves];
  __shared__ Border borders[2];
  __shared__ int arrived;

  const int tid = static_cast<int>(threadIdx.x);
  const int n_blocks = static_cast<int>(gridDim.x);

  // Every block sums the sequences' weights and finds its share's two borders.
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0;
  Seq s = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    s = load_seq(p, b);
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
  if (tid < 2) borders[tid].b = p.batch;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < (tid >> 6)) before += wave_weight[w];
    total += wave_weight[w];
  }
  before -= mine;
  const int64_t share = max(floor_div(total, n_blocks) + 1, static_cast<int64_t>(kMinShareKeys));
  // Neighbouring shares read the same keys, so they go to one XCD (blocks are
  // dealt to the 8 XCDs in turn).
  const int active = static_cast<int>(floor_div(total, share)) + 1;
  const int per_xcd = (min(active, n_blocks) + 7) / 8;
  const int blk = static_cast<int>(blockIdx.x);
  const int w = blk < 8 * per_xcd ? (blk & 7) * per_xcd + (blk >> 3) : blk;
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int64_t at = (w + side) * share;
    if (at < before || at >= before + mine) continue;
    int64_t from = before;
    for (int b = b0; b < b1; ++b) {
      if (per > 1) s = load_seq(p, b);
      const Tiles t = tiles_of(p, s.n);
      const int64_t whole = weight_before(p, s, t, t.count);
      if (at < from + whole * p.kv_heads) {
        borders[side] = border_in(p, s, t, b, whole, from, at);
        break;
      }
      from += whole * p.kv_heads;
    }
  }
  __syncthreads();
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  int b = uniform(borders[0].b), kvh = uniform(borders[0].kvh), tile = uniform(borders[0].tile);
  int kt = uniform(borders[0].kt);
  s.t0 = uniform(borders[0].s.t0);
  s.n = uniform(borders[0].s.n);
  s.p0 = uniform(borders[0].s.p0);
  int64_t from = borders[0].from;
  const int end_b = uniform(borders[1].b), end_kvh = uniform(borders[1].kvh);
  const int end_tile = uniform(borders[1].tile), end_kt = uniform(borders[1].kt);

  const unsigned ring = lds_addr(ring_mem);
  Tiles t = tiles_of(p, s.n);
  while (b < p.batch) {
    if (tile >= t.count) {  // next K/V head or sequence
      tile = 0;
      kt = 0;
      if (t.count == 0 || ++kvh >= p.kv_heads) {
        from += weight_before(p, s, t, t.count) * p.kv_heads;
        kvh = 0;
        ++b;
        if (b >= p.batch) break;
        s = load_seq(p, b);
        s.t0 = uniform(s.t0);
        s.n = uniform(s.n);
        s.p0 = uniform(s.p0);
        t = tiles_of(p, s.n);
      }
      if (b > end_b) break;
      continue;
    }
    const bool last = b == end_b && kvh == end_kvh && tile == end_tile;
    Item it;
    it.end = key_end(p, s, t, tile);
    const int tiles = key_tiles(it.end);
    it.kt0 = kt;
    it.kt1 = last ? min(end_kt, tiles) : tiles;
    it.t0 = s.t0 + tile * t.tokens;
    it.n = min(t.tokens, s.n - tile * t.tokens);
    it.p0 = s.p0 + tile * t.tokens;
    it.kvh = kvh;
    it.table = (uniform_table)(reinterpret_cast<uintptr_t>(
        p.page_table + static_cast<int64_t>(b) * p.max_pages));
    // A whole item (also one that sees no key) is written out; a part leaves a partial.
    const bool whole = it.kt0 == 0 && it.kt1 == tiles && !(last && end_kt < tiles) &&
                       !(last && tiles == 0);
    if (whole || it.kt1 > it.kt0) {
      it.slot = whole ? -1 : 2 * w + (it.kt0 == 0 ? 1 : 0);
      if (it.n * p.group <= kNarrowRows)
        narrow_item<T, D>(p, it, ring, reinterpret_cast<float *>(ring_mem), ml_mem);
      else
        wide_item<T, D>(p, it, ring);
    }
    if (!whole && it.kt1 > it.kt0) {
      const int64_t x0 = from + kvh * weight_before(p, s, t, t.count) + weight_before(p, s, t, tile);
      const int64_t x1 = x0 + weight_before(p, s, t, tile + 1) - weight_before(p, s, t, tile);
      const Pieces pc = pieces_of(x0, x1, tiles, share);
      // The partial is stored before it is counted; the block that counts last sets the
      // counter back to zero for the next call.
      wait_loads<0>();
      __syncthreads();
      if (tid == 0) {
        unsigned *counter = p.counters + pc.first;
        const unsigned n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT);
        arrived = static_cast<int>(n) + 1;
        if (arrived == pc.count)
          __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (arrived == pc.count) {
        if (it.n * p.group <= kNarrowRows) join_narrow<T, D>(p, it, pc);
        else join_wide<T, D>(p, it, pc);
      }
      __syncthreads();
    }
    if (last) break;
    ++tile;
    kt = 0;
  }

  // Outputs of packed rows that belong to no sequence are zero.
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

// Zeroes the arrival counters of a call whose stream has no counter slot.
__global__ void zero_counters_kernel(unsigned *counters, int n) {
  const int i = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
  if (i < n) counters[i] = 0;
}

int attend_blocks() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  return 2 * device_cu_count(dev);
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
  const size_t n = static_cast<size_t>(attend_blocks());
  return counter_bytes(n) +
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
  p.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                         counter_bytes(static_cast<size_t>(n_blocks)));
  // Arrival counters: the stream's own, zero between calls, or, where it has no slot,
  // the workspace's, zeroed by a launch of their own.
  p.counters = merge_counters(stream, static_cast<size_t>(n_blocks));
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
