// Rotary positions, and the write of a ragged batch's new tokens into a paged
// K/V cache with the rotation of its queries and keys fused in.
//
// No reference counterpart: its callers rotate q and k before prefill / decode
// and write their own cache (README.md:9-13 of shrvan30/flash-attention-cuda).
//
// Mathematics. Pair i of a row at position p turns by theta = p w_i:
//   (a, c) -> factor * (a cos theta - c sin theta, a sin theta + c cos theta);
// the gradient is the transposed matrix, i.e. the turn by -theta with the same
// factor. Pair i is dims (i, i + R/2) (halves) or (2i, 2i + 1) (interleaved) of
// the first R dims; dims from R on are copied.
//   theta is reduced in 64 bits: p w / (2 pi) has as many integer turns as the
//   position is far (2^20 at p = 2^23, w = 1), so in 32 bits a far position
//   would keep only a few bits of its angle. The fraction of a turn, in
//   [-1/2, 1/2], then needs no more than 32 bits; sine and cosine are taken of
//   it in 32 bits, and the result is rounded once to the tensor's type.
//
// Work per thread: 16 dims of a row, as two 16-byte pieces: 8 pairs (halves:
// dims [8u, +8) and [R/2 + 8u, +8); interleaved: dims [16u, +16)), or 16 dims to
// copy. The eight sines and cosines serve every head the thread loops over.
//
// What bounds it: HBM, or for a step's few rows the launch and its chain of loads (us per
// call among others, distinct inputs; floor: bytes at 6.25 TB/s, an elementwise pass over 1 GiB):
//   rope B8 H32 S4096 D128 bf16, 537 MB            117     (floor 85.9; one input over and over
//                                                  83, part of it then lies in the last cache)
//   rope_backward B4 H12 S4096 D64 bf16, 50 MB      10.1   (8.1)
//   append 6144 tokens H32/8 D128 bf16, 151 MB      25.5   (24.2)
//   in a graph of calls: rope of one token 2.9, append of 32 tokens 3.4

#include "fa_internal.h"

namespace fa {
namespace {

constexpr int kRopeThreads = 256;

template <typename T>
struct Vec8;
template <>
struct Vec8<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Vec8<__bf16> {
  typedef __bf16 type __attribute__((ext_vector_type(8)));
};

// cos and sin (times factor) of the 8 pairs [8 u, 8 u + 8) at position p.
struct Turns {
  float c[8], s[8];
};
__device__ __forceinline__ void turns_of(const double *__restrict__ inv_freq, int u, double p,
                                         float factor, Turns &t) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double turn = p * (inv_freq[8 * u + i] * 0.15915494309189533577);  // 1 / (2 pi)
    const float frac = static_cast<float>(turn - rint(turn));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    t.c[i] = cs * factor;
    t.s[i] = sn * factor;
  }
}

// Offsets of a thread's two 16-byte pieces in a row, and whether it rotates.
struct Piece {
  int first, second;
  bool turned;
};
__device__ __forceinline__ Piece piece_of(int u, int rotary, bool interleaved) {
  Piece p;
  p.turned = u < rotary / 16;
  p.first = (p.turned && !interleaved) ? 8 * u : 16 * u;
  p.second = (p.turned && !interleaved) ? 8 * u + rotary / 2 : 16 * u + 8;
  return p;
}

template <typename T>
__device__ __forceinline__ void turn(typename Vec8<T>::type &x, typename Vec8<T>::type &y,
                                     const Turns &t, bool interleaved) {
  float a[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = static_cast<float>(x[i]);
    a[8 + i] = static_cast<float>(y[i]);
  }
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = a[2 * i] * t.c[i] - a[2 * i + 1] * t.s[i];
      const float o = a[2 * i] * t.s[i] + a[2 * i + 1] * t.c[i];
      a[2 * i] = e;
      a[2 * i + 1] = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = a[i] * t.c[i] - a[8 + i] * t.s[i];
      const float o = a[i] * t.s[i] + a[8 + i] * t.c[i];
      a[i] = e;
      a[8 + i] = o;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = static_cast<T>(a[i]);
    y[i] = static_cast<T>(a[8 + i]);
  }
}

struct RopeParams {
  const void *x;
  void *out;
  const int32_t *positions;
  const double *inv_freq;
  int64_t x_batch, x_head, x_row;  // strides of x in elements
  int64_t pos_batch;               // stride of positions (0: one row for every sequence)
  unsigned units;                  // batch * seq * head_dim / 16, under 2^31
  int heads, seq, head_dim, rotary, heads_per_thread;
  float factor;
  bool interleaved, backward;
};

template <typename T>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeParams p) {
  typedef typename Vec8<T>::type V;
  const unsigned i = blockIdx.x * kRopeThreads + threadIdx.x;
  if (i >= p.units) return;
  const int row_shift = p.head_dim == 64 ? 2 : 3;
  const int u = static_cast<int>(i & ((1u << row_shift) - 1));
  const unsigned token = i >> row_shift;
  const int64_t b = token / static_cast<unsigned>(p.seq);
  const int n = static_cast<int>(token - static_cast<unsigned>(b) * p.seq);
  const int h0 = static_cast<int>(blockIdx.y) * p.heads_per_thread;
  const int h1 = min(h0 + p.heads_per_thread, p.heads);
  const Piece at = piece_of(u, p.rotary, p.interleaved);
  Turns t;
  if (at.turned) {
    const double pos = static_cast<double>(p.positions[b * p.pos_batch + n]);
    turns_of(p.inv_freq, u, p.backward ? -pos : pos, p.factor, t);
  }
  const T *x = static_cast<const T *>(p.x) + b * p.x_batch + n * p.x_row;
  T *o = static_cast<T *>(p.out) + (b * p.heads * p.seq + n) * p.head_dim;
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const T *xr = x + h * p.x_head;
    T *out = o + static_cast<int64_t>(h) * p.seq * p.head_dim;
    V a = *reinterpret_cast<const V *>(xr + at.first);
    V c = *reinterpret_cast<const V *>(xr + at.second);
    if (at.turned) turn<T>(a, c, t, p.interleaved);
    // Plain stores: non-temporal ones leave less of the output in a cache for the call that
    // reads it. Alone 112.5 us for 115.1 (268 MB, D128) or 115.3 for 113.5 (D64), with an
    // elementwise reader behind it 214.7 for 202.6 and 214.4 for 202.4; smaller outputs alike
    // (67 MB, D128: 22.6 for 28.5 alone, 55.1 for 47.7 with the reader).
    *reinterpret_cast<V *>(out + at.first) = a;
    *reinterpret_cast<V *>(out + at.second) = c;
  }
}

// Sequence of a packed token: the number of entries of bounds[1..batch] that
// are <= token (batch: behind the last sequence). A step of one token per
// sequence holds token t in sequence t, which two loads confirm; otherwise a
// binary search. Any contents of `bounds` give a value in [0, batch].
__device__ __forceinline__ int sequence_of(const int32_t *__restrict__ bounds, int batch,
                                           int token) {
  if (token < batch && bounds[token] == token && bounds[token + 1] == token + 1) return token;
  int lo = 0, hi = batch;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (bounds[mid + 1] <= token) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kRopeThreads) void append_paged_kernel(const AppendPagedParams p) {
  typedef typename Vec8<T>::type V;
  const unsigned i = blockIdx.x * kRopeThreads + threadIdx.x;
  const int row_shift = p.head_dim == 64 ? 2 : 3;
  const int u = static_cast<int>(i & ((1u << row_shift) - 1));
  const int t = static_cast<int>(i >> row_shift);
  if (t >= p.tokens) return;
  const int64_t token = t;
  const Piece at = piece_of(u, p.rotary, p.interleaved);
  const int h0 = static_cast<int>(blockIdx.y) * p.heads_per_thread;
  const int h1 = min(h0 + p.heads_per_thread, p.q_heads + 2 * p.kv_heads);

  // Tokens in front of the first sequence's count as its own there.
  const int b = sequence_of(p.cu_tokens, p.batch, t);
  const bool live = b < p.batch && t >= p.cu_tokens[b];
  int64_t pos = 0;
  int64_t row = -1;  // row of the token in the page pool, counted over (page, row) pairs
  if (live) {
    pos = static_cast<int64_t>(p.seq_lens[b]) - p.cu_tokens[b + 1] + t;
    if (pos >= 0 && (pos >> p.page_shift) < p.max_pages) {
      const int page = p.page_table[static_cast<int64_t>(b) * p.max_pages + (pos >> p.page_shift)];
      if (page >= 0 && page < p.num_pages)
        row = ((static_cast<int64_t>(page) * p.kv_heads) << p.page_shift) +
              (pos & ((1 << p.page_shift) - 1));
    }
  }
  Turns turns;
  if (at.turned) turns_of(p.inv_freq, u, static_cast<double>(pos), p.factor, turns);

#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    // Heads are numbered q, then k, then v.
    const int kh = h - p.q_heads, vh = kh - p.kv_heads;
    const T *src;
    T *dst;
    if (kh < 0) {
      src = static_cast<const T *>(p.q) + token * p.q_token + h * p.q_head;
      dst = static_cast<T *>(p.q_out) + (token * p.q_heads + h) * p.head_dim;
    } else {
      const int head = vh < 0 ? kh : vh;
      src = vh < 0 ? static_cast<const T *>(p.k) + token * p.k_token + head * p.k_head
                   : static_cast<const T *>(p.v) + token * p.v_token + head * p.v_head;
      dst = static_cast<T *>(vh < 0 ? p.k_pages : p.v_pages) +
            (row + (static_cast<int64_t>(head) << p.page_shift)) * p.head_dim;
      if (row < 0) continue;
    }
    V a = *reinterpret_cast<const V *>(src + at.first);
    V c = *reinterpret_cast<const V *>(src + at.second);
    if (vh < 0 && at.turned) turn<T>(a, c, turns, p.interleaved);
    if (!live) a = c = V{};  // a query row outside every sequence
    // Non-temporal stores do not claim L2 lines that the loads want: 6144 tokens H32/8 D128
    // 34.7 -> 26.4 us, few tokens alike. With attend_paged behind it, which finds less of q in
    // the caches, those 6144 tokens take 173.7 us for 168.7, 128 single tokens 33.8 for 34.7.
    __builtin_nontemporal_store(a, reinterpret_cast<V *>(dst + at.first));
    __builtin_nontemporal_store(c, reinterpret_cast<V *>(dst + at.second));
  }
}

// Heads one thread takes: up to 8, since 8 sines and cosines cost as many instructions as
// about 6 heads' loads, products and stores, fewer while the launch has under kFill threads
// per CU (B2 H14 S1733 D64: 5.7 us at 2048, 5.2 at 512; 466 tokens of H32/8 D128: 7.9, 6.8,
// and 9.2 at 128).
constexpr int kFill = 512;
int heads_per_thread(int64_t units, int heads) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const int64_t want = static_cast<int64_t>(device_cu_count(dev)) * kFill;
  int n = 8;
  while (n > 1 && units * ((heads + n - 1) / n) < want) n /= 2;
  return n;
}

}  // namespace

int launch_rope(const void *x, void *out, const int32_t *positions, const double *inv_freq,
                bool bf16, int batch, int heads, int seq, int head_dim, int64_t x_batch,
                int64_t x_head, int64_t x_row, int64_t pos_batch, int rotary, bool interleaved,
                float factor, bool backward, hipStream_t stream) {
  RopeParams p;
  p.x = x;
  p.out = out;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.x_batch = x_batch;
  p.x_head = x_head;
  p.x_row = x_row;
  p.pos_batch = pos_batch;
  p.units = static_cast<unsigned>(batch) * static_cast<unsigned>(seq) * (head_dim / 16);
  p.heads = heads;
  p.seq = seq;
  p.head_dim = head_dim;
  p.rotary = rotary;
  p.heads_per_thread = heads_per_thread(p.units, heads);
  p.factor = factor;
  p.interleaved = interleaved;
  p.backward = backward;
  const dim3 grid(static_cast<unsigned>((p.units + kRopeThreads - 1) / kRopeThreads),
                  static_cast<unsigned>((heads + p.heads_per_thread - 1) / p.heads_per_thread));
  auto *kernel = bf16 ? rope_kernel<__bf16> : rope_kernel<_Float16>;
  hipLaunchKernelGGL(kernel, grid, dim3(kRopeThreads), 0, stream, p);
  return check_hip(hipGetLastError(), "rope_kernel launch");
}

int launch_append_paged(AppendPagedParams p, bool bf16, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(p.tokens) * (p.head_dim / 16);
  const int heads = p.q_heads + 2 * p.kv_heads;
  p.heads_per_thread = heads_per_thread(units, heads);
  const dim3 grid(static_cast<unsigned>((units + kRopeThreads - 1) / kRopeThreads),
                  static_cast<unsigned>((heads + p.heads_per_thread - 1) / p.heads_per_thread));
  if (bf16) hipLaunchKernelGGL(append_paged_kernel<__bf16>, grid, dim3(kRopeThreads), 0, stream, p);
  else hipLaunchKernelGGL(append_paged_kernel<_Float16>, grid, dim3(kRopeThreads), 0, stream, p);
  return check_hip(hipGetLastError(), "append_paged_kernel launch");
}

}  // namespace fa
