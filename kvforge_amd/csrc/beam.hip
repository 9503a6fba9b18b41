// Beam search between two forward passes: which continuations of a request's beams live on, and what they own
// following them.
//
// Selection.  With logits l of a beam's row and the beam's running score S, candidate (beam, token) scores
//   S + (l - m) - log(sum_t exp(l_t - m)),   m = max_t l_t,
// and the `count` best of a request are wanted, best first, equal scores by the lower beam, then the lower token.
// Logits that are NaN or -inf are no candidates and weigh nothing, +inf counts as the largest finite number, and
// beams whose score is not finite are passed over unread.
//
//   1. `beam_pieces_kernel`, a workgroup a piece of a row: the piece stays in registers (E logits a lane), so the row is
//      read once.  Maximum, sum of exponentials, and the piece's `count` best, sorted.  They are found by a bound: of the
//      64 largest logits of a wave's lanes, the `count`-th largest is settled bit by bit with ballots; at least `count`
//      logits reach it, and seldom many more.  What reaches the best of the four waves' bounds goes to a list in LDS,
//      where every entry counts those ahead of it: its place.  (Logits equal to the bound are taken in the order of their tokens, no
//      more than `count` a wave, so the list holds whatever the logits are.)
//   2. `beam_best_kernel`, a workgroup a request: joins the sums of a row's pieces in 64 bits (candidates of different
//      beams may lie closer than 32 bits tell apart: their order is the sums' order), then merges the sorted lists of all rows,
//      the lists of a wave side by side: of two sorted lists the larger of a[i] and b[count - 1 - i] are the best of both, and
//      log2(count) exchanges sort them again.
//
// Reordering: see `beam_reorder_kernel`.
#include "common.h"

namespace {
constexpr int THREADS = 256, NWAVES = THREADS / KVF_WAVE;
constexpr int MAX_COUNT = 64;

// The order of finite numbers as unsigned integers; 0 stands below all of them ("no candidate").
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// exp(x) for x <= 0 to about 2^-24, without the bias that one rounded constant gives all terms of a sum: the product with
// log2(e) is carried in two parts, the second of which joins behind the hardware's base-2 exponential.
__device__ __forceinline__ float exp_unbiased(float x) {
  constexpr float L = 1.44269504088896340736f;
  constexpr float L_LO = static_cast<float>(1.44269504088896340736 - static_cast<double>(L));
  constexpr float LN2 = 0.693147180559945f;
  x = fmaxf(x, -200.f);            // -inf too: nothing in 32 bits
  const float hi = x * L;
  const float lo = fmaf(x, L, -hi) + x * L_LO;
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, lo * LN2, e);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = KVF_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, KVF_WAVE);
  return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int o = KVF_WAVE / 2; o > 0; o >>= 1) {
    const uint32_t n = __shfl_xor(v, o, KVF_WAVE);
    v = n > v ? n : v;
  }
  return v;
}

// The `count`-th largest of 64 lanes' keys (0 where fewer are above 0).
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t key, int count) {
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t want = found | (1u << bit);
    if (__popcll(__ballot(key >= want)) >= count) found = want;
  }
  return found;
}

// 16 bytes of logits at p[0..], as keys; places outside [0, n) give 0.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  }
};
template <> struct Chunk<bf16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[8]) { load8(p, v); }
};

__device__ __forceinline__ bool alive(float score) { return fabsf(score) <= 3.402823466e38f; }

struct PieceArgs {
  long stride;          // elements from one row of logits to the next
  int rows, vocab, count, pieces, piece;   // `piece`: elements of a piece, a multiple of THREADS * Chunk::N
};

// sums[row][piece] = (sum of exponentials, their reference), values/tokens[row][piece][count]: sorted, token -1 behind the last.
template <typename T, int E>
__global__ __launch_bounds__(THREADS) void beam_pieces_kernel(const T* __restrict__ logits, const float* __restrict__ scores,
                                                              double2* __restrict__ sums, float* __restrict__ values,
                                                              int* __restrict__ tokens, PieceArgs a) {
  constexpr int N = Chunk<T>::N, CHUNKS = E / N;
  extern __shared__ unsigned long long list[];   // (key, ~token) of what reaches the bound
  __shared__ uint32_t bound_of[NWAVES];
  __shared__ float max_of[NWAVES];
  __shared__ double sum_of[NWAVES];
  __shared__ int n_list;
  const int tid = threadIdx.x, lane = tid % KVF_WAVE, wave = tid / KVF_WAVE;
  const int row = blockIdx.y, piece = blockIdx.x;
  const size_t at = static_cast<size_t>(row) * a.pieces + piece;
  float* out_v = values + at * a.count;
  int* out_t = tokens + at * a.count;
  if (!alive(scores[row])) {       // the whole workgroup: the merge passes such rows over
    return;
  }
  const T* x = logits + row * a.stride;
  // chunks lie on 16 bytes of memory: element e of the row is place e + skip of its first chunk's line
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const int lo = piece * a.piece - skip;        // the piece's first element (below 0 in front of the row)
  const int hi = min(lo + a.piece, a.vocab);
  float v[CHUNKS][N];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int e = lo + (c * THREADS + tid) * N;
    if (e >= 0 && e + N <= hi) {
      Chunk<T>::load(x + e, v[c]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[c][i] = e + i >= 0 && e + i < hi ? Elem<T>::load(x + e + i) : -INFINITY;
    }
  }
  if (tid == 0) n_list = 0;
  // NaN becomes -inf (fmaxf gives the other operand), +inf the largest finite number
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[c][i] = fminf(fmaxf(v[c][i], -INFINITY), 3.402823466e38f) + 0.f;     // (-0 equals 0)
      mx = fmaxf(mx, v[c][i]);
    }
  const uint32_t lane_key = mx > -INFINITY ? order_key(mx) : 0u;
  const uint32_t wave_bound = kth_of_lanes(lane_key, a.count);
  const float wmx = wave_max(mx);
  if (lane == 0) {
    bound_of[wave] = wave_bound;
    max_of[wave] = wmx;
  }
  __syncthreads();
  uint32_t bound = 0;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) {
    bound = bound_of[w] > bound ? bound_of[w] : bound;
    m = fmaxf(m, max_of[w]);
  }
  // what is ahead of the bound, and what equals it in the order of the tokens
  const unsigned long long below = (1ull << lane) - 1ull;
  const float least = bound ? key_value(bound) : -INFINITY;
  int ties = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= v[c][i] >= least && v[c][i] > -INFINITY;
    if (!__ballot(any)) continue;
    const int e = lo + (c * THREADS + tid) * N;
    unsigned long long same[N];
    int before = ties, all = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool ahead = v[c][i] > least;
      const unsigned long long who = __ballot(ahead);
      if (who) {
        int base = 0;
        if (lane == 0) base = atomicAdd(&n_list, static_cast<int>(__popcll(who)));
        base = __shfl(base, 0, KVF_WAVE);
        if (ahead)
          list[base + __popcll(who & below)] = static_cast<unsigned long long>(order_key(v[c][i])) << 32 | static_cast<uint32_t>(~(e + i));
      }
      same[i] = __ballot(v[c][i] == least && least > -INFINITY);
      before += __popcll(same[i] & below);
      all += __popcll(same[i]);
    }
    if (all && ties < a.count) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool mine = same[i] >> lane & 1ull;
        const unsigned long long who = __ballot(mine && before < a.count);
        if (who) {
          int base = 0;
          if (lane == 0) base = atomicAdd(&n_list, static_cast<int>(__popcll(who)));
          base = __shfl(base, 0, KVF_WAVE);
          if (mine && before < a.count)
            list[base + __popcll(who & below)] = static_cast<unsigned long long>(bound) << 32 | static_cast<uint32_t>(~(e + i));
        }
        before += mine;
      }
    }
    ties += all;
  }
  // the sum, while the list's entries arrive
  double s = 0.0;
  if (m > -INFINITY) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) s += static_cast<double>(exp_unbiased(v[c][i] - m));
  }
  s = wave_sum64(s);
  if (lane == 0) sum_of[wave] = s;
  __syncthreads();
  const int n = n_list;
  for (int i = tid; i < n; i += THREADS) {
    const unsigned long long mine = list[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += list[j] > mine;
    if (place < a.count) {
      out_v[place] = key_value(static_cast<uint32_t>(mine >> 32));
      out_t[place] = static_cast<int>(~static_cast<uint32_t>(mine));
    }
  }
  for (int i = n + tid; i < a.count; i += THREADS) {
    out_v[i] = -INFINITY;
    out_t[i] = -1;
  }
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < NWAVES; ++w) total += sum_of[w];
    sums[at] = make_double2(total, static_cast<double>(m));
  }
}

// An entry of a sorted list: score, and what tells equal scores apart (lower first): the beam in the upper 16 bits, then the
// logit, largest first (scores of a beam may be equal in 64 bits though its logits are not), then the place in the beam's
// lists, which is in the order of the tokens.
struct Entry {
  double score;
  unsigned long long tie;
};
constexpr unsigned long long NOBODY = ~0ull;
__device__ __forceinline__ bool ahead(const Entry& a, const Entry& b) {
  return a.score > b.score || (a.score == b.score && a.tie < b.tie);
}
template <typename T> __device__ __forceinline__ T from_lane(T v, int lane) { return __shfl(v, lane, KVF_WAVE); }
__device__ __forceinline__ Entry entry_of(const Entry& e, int lane) { return {from_lane(e.score, lane), from_lane(e.tie, lane)}; }

// The best L of two sorted lists of L that lie in groups of L lanes (L a power of two), sorted.
template <int L> __device__ __forceinline__ Entry merge_lists(Entry mine, Entry other_reversed, int lane) {
  Entry e = ahead(mine, other_reversed) ? mine : other_reversed;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const Entry n = entry_of(e, lane ^ o);
    const bool first = (lane & o) == 0;
    if (first == ahead(n, e)) e = n;
  }
  return e;
}

struct BestArgs {
  int rows, requests, count, pieces;
};

// row_of[row] = (reference, S - log(sum)); then the request's candidates.  L: `count` rounded up to a power of two.
template <int L>
__global__ __launch_bounds__(THREADS) void beam_best_kernel(const float* __restrict__ scores, const int* __restrict__ cu_beams,
                                                            const double2* __restrict__ sums, const float* __restrict__ values,
                                                            const int* __restrict__ tokens, double2* __restrict__ row_of,
                                                            float* __restrict__ out_scores, int* __restrict__ out_beams,
                                                            int* __restrict__ out_tokens, BestArgs a) {
  __shared__ double list_s[NWAVES][L];
  __shared__ unsigned long long list_t[NWAVES][L];
  const int tid = threadIdx.x, lane = tid % KVF_WAVE, wave = tid / KVF_WAVE;
  const int request = blockIdx.x;
  const int first = min(max(cu_beams[request], 0), a.rows);
  const int beams = min(max(cu_beams[request + 1], first), a.rows) - first;
  for (int b = wave; b < beams; b += NWAVES) {
    const int row = first + b;
    const float score = scores[row];
    double m = -INFINITY, s = 0.0;
    if (alive(score)) {
      const double2* p = sums + static_cast<size_t>(row) * a.pieces;
      for (int i = lane; i < a.pieces; i += KVF_WAVE) m = fmax(m, p[i].y);
#pragma unroll
      for (int o = KVF_WAVE / 2; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o, KVF_WAVE));
      if (m > -INFINITY)
        for (int i = lane; i < a.pieces; i += KVF_WAVE) s += p[i].x * exp(p[i].y - m);
      s = wave_sum64(s);
    }
    if (lane == 0) row_of[row] = make_double2(m, s > 0.0 ? static_cast<double>(score) - log(s) : -INFINITY);
  }
  __syncthreads();
  const int lists = beams * a.pieces;
  constexpr int SIDE = KVF_WAVE / L;       // lists side by side in a wave
  const int group = lane / L, at = lane % L;
  auto entry = [&](int l, int i) {         // entry i of list l of the request
    Entry e{-INFINITY, NOBODY};
    if (l < lists && i < a.count) {
      const int beam = l / a.pieces, row = first + beam;
      const size_t from = (static_cast<size_t>(first) * a.pieces + l) * a.count + i;
      const double2 r = row_of[row];
      if (r.y > -INFINITY && tokens[from] >= 0) {
        e.score = (static_cast<double>(values[from]) - r.x) + r.y;
        e.tie = static_cast<unsigned long long>(beam) << 48 | static_cast<unsigned long long>(~order_key(values[from])) << 16 |
                static_cast<unsigned long long>((l - beam * a.pieces) * a.count + i);
      }
    }
    return e;
  };
  int l = wave * SIDE + group;
  Entry best = entry(l, at);
  for (l += NWAVES * SIDE; l - group < lists; l += NWAVES * SIDE) best = merge_lists<L>(best, entry(l, L - 1 - at), lane);
#pragma unroll
  for (int o = L; o < KVF_WAVE; o <<= 1) {      // the groups of the wave
    const Entry other = entry_of(best, (lane ^ o) ^ (L - 1));
    best = merge_lists<L>(best, other, lane);
  }
  if (lane < L) {
    list_s[wave][lane] = best.score;
    list_t[wave][lane] = best.tie;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < NWAVES; ++w) {
    const Entry other{list_s[w][L - 1 - at], list_t[w][L - 1 - at]};
    best = merge_lists<L>(best, other, lane);
  }
  if (lane < a.count) {
    const bool there = best.tie != NOBODY;
    const int beam = static_cast<int>(best.tie >> 48);
    const size_t to = static_cast<size_t>(request) * a.count + lane;
    out_scores[to] = there ? static_cast<float>(best.score) : -INFINITY;
    out_beams[to] = there ? beam : -1;
    out_tokens[to] = there ? tokens[static_cast<size_t>(first + beam) * a.pieces * a.count + (best.tie & 0xffffull)] : -1;
  }
}

template <typename T, int E>
int pieces_launch(const void* logits, const float* scores, double2* sums, float* values, int* tokens, const PieceArgs& a, hipStream_t stream) {
  // what is strictly ahead of the bound lies in fewer than `count` lanes of every wave; equals: `count` a wave
  const size_t lds = static_cast<size_t>(NWAVES) * ((a.count - 1) * E + a.count) * sizeof(unsigned long long);
  beam_pieces_kernel<T, E><<<dim3(a.pieces, a.rows), THREADS, lds, stream>>>(static_cast<const T*>(logits), scores, sums, values, tokens, a);
  return kvf_last_error();
}
}  // namespace

// logits [rows][stride] of `vocab` (bf16: 0 fp32, 1 bf16); scores [rows]; cu_beams [requests + 1]; out_* [requests][count].
// Workspace: sums [rows][pieces][2] and row_of [rows][2] in 64 bits, values/tokens [rows][pieces][count].  piece: elements of a
// piece, 256 times 8 or 32.
KVF_EXPORT int kvf_beam_select(int bf16, const void* logits, long stride, int rows, int vocab, const float* scores,
                               const int* cu_beams, int requests, int count, int pieces, int piece, void* sums, void* row_of,
                               float* values, int* tokens, float* out_scores, int* out_beams, int* out_tokens,
                               hipStream_t stream) {
  if (count < 1 || count > MAX_COUNT || rows < 0 || rows > 65535 || vocab < 1 || pieces < 1 || requests < 0 ||
      static_cast<long>(pieces) * count > 65536)
    return static_cast<int>(hipErrorInvalidValue);
  if (piece != THREADS * 8 && piece != THREADS * 32) return static_cast<int>(hipErrorInvalidValue);
  if (requests == 0) return 0;
  // a row may begin up to 15 bytes into its first chunk
  if (static_cast<long>(pieces) * piece < static_cast<long>(vocab) + (bf16 ? 7 : 3)) return static_cast<int>(hipErrorInvalidValue);
  if (rows) {
    const PieceArgs a{stride, rows, vocab, count, pieces, piece};
    auto* s = static_cast<double2*>(sums);
    int rc;
    if (bf16)
      rc = piece == THREADS * 8 ? pieces_launch<bf16_t, 8>(logits, scores, s, values, tokens, a, stream)
                                : pieces_launch<bf16_t, 32>(logits, scores, s, values, tokens, a, stream);
    else
      rc = piece == THREADS * 8 ? pieces_launch<float, 8>(logits, scores, s, values, tokens, a, stream)
                                : pieces_launch<float, 32>(logits, scores, s, values, tokens, a, stream);
    if (rc) return rc;
  }
  const BestArgs b{rows, requests, count, pieces};
  const auto* s = static_cast<const double2*>(sums);
  auto* r = static_cast<double2*>(row_of);
#define KVF_BEST(L) beam_best_kernel<L><<<requests, THREADS, 0, stream>>>(scores, cu_beams, s, values, tokens, r, out_scores, out_beams, out_tokens, b)
  if (count <= 4) KVF_BEST(4);
  else if (count <= 8) KVF_BEST(8);
  else if (count <= 16) KVF_BEST(16);
  else if (count <= 32) KVF_BEST(32);
  else KVF_BEST(64);
#undef KVF_BEST
  return kvf_last_error();
}

namespace {
// What a set of tensors is made of: tensor t has rows of `bytes` bytes, `stride` bytes apart, read and written `unit` bytes at a time.
struct RowsOf {
  char* base;
  long stride, bytes, unit;
};
struct Tile {
  int tensor, number;    // tile `number` of the tensor's rows: TILE_BYTES of them
};
constexpr int TILE_BYTES = THREADS * 16;

template <typename U> struct Words { static constexpr int N = 16 / sizeof(U); };

// A workgroup takes a tile of bytes of one tensor, of all W rows of a request: a lane's bytes of every row that moves are in its
// registers before it writes any of them, and no other lane touches them, so rows may change places in any way (swaps and rings
// too) without memory beside them.
template <typename U, int W>
__device__ __forceinline__ void move_rows(const RowsOf& t, int number, int rows, int beams, const int* __restrict__ slots,
                                          const int* __restrict__ parents) {
  constexpr int N = Words<U>::N;
  U v[W][N];
  const long from = static_cast<long>(number) * TILE_BYTES + threadIdx.x * sizeof(U);
  int to[W];
#pragma unroll
  for (int b = 0; b < W; ++b) {
    to[b] = -1;
    if (b >= beams) continue;
    const int p = parents[b];
    if (p == b || p < 0 || p >= beams) continue;
    const int dst = slots[b], src = slots[p];
    if (dst < 0 || dst >= rows || src < 0 || src >= rows || src == dst) continue;
    to[b] = dst;
    const char* row = t.base + src * t.stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const long o = from + static_cast<long>(i) * THREADS * sizeof(U);
      if (o < t.bytes) v[b][i] = *reinterpret_cast<const U*>(row + o);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // all read before any is written
#pragma unroll
  for (int b = 0; b < W; ++b) {
    if (to[b] < 0) continue;
    char* row = t.base + to[b] * t.stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const long o = from + static_cast<long>(i) * THREADS * sizeof(U);
      if (o < t.bytes) *reinterpret_cast<U*>(row + o) = v[b][i];
    }
  }
}

template <int W>
__global__ __launch_bounds__(THREADS) void beam_reorder_kernel(const RowsOf* __restrict__ tensors, const Tile* __restrict__ tiles,
                                                               int rows, int beams, const int* __restrict__ slots,
                                                               const int* __restrict__ parents) {
  const Tile tile = tiles[blockIdx.x];
  const RowsOf t = tensors[tile.tensor];
  slots += static_cast<size_t>(blockIdx.y) * beams;
  parents += static_cast<size_t>(blockIdx.y) * beams;
  if (t.unit == 16) move_rows<uint4, W>(t, tile.number, rows, beams, slots, parents);
  else if (t.unit == 8) move_rows<uint2, W>(t, tile.number, rows, beams, slots, parents);
  else if (t.unit == 4) move_rows<uint32_t, W>(t, tile.number, rows, beams, slots, parents);
  else move_rows<uint16_t, W>(t, tile.number, rows, beams, slots, parents);
}
}  // namespace

KVF_EXPORT int kvf_beam_tile_bytes() { return TILE_BYTES; }

// tensors: RowsOf (four 64-bit numbers) each; tiles: (tensor, number) each; slots, parents [requests][beams].
KVF_EXPORT int kvf_beam_reorder(const void* tensors, const void* tiles, int n_tiles, int rows, int requests, int beams,
                                const int* slots, const int* parents, hipStream_t stream) {
  if (beams < 1 || beams > 32 || requests < 0 || requests > 65535 || n_tiles < 0 || rows < 0) return static_cast<int>(hipErrorInvalidValue);
  if (requests == 0 || n_tiles == 0 || beams == 1) return 0;
  const auto* t = static_cast<const RowsOf*>(tensors);
  const auto* l = static_cast<const Tile*>(tiles);
  const dim3 grid(n_tiles, requests);
  if (beams <= 4) beam_reorder_kernel<4><<<grid, THREADS, 0, stream>>>(t, l, rows, beams, slots, parents);
  else if (beams <= 8) beam_reorder_kernel<8><<<grid, THREADS, 0, stream>>>(t, l, rows, beams, slots, parents);
  else if (beams <= 16) beam_reorder_kernel<16><<<grid, THREADS, 0, stream>>>(t, l, rows, beams, slots, parents);
  else beam_reorder_kernel<32><<<grid, THREADS, 0, stream>>>(t, l, rows, beams, slots, parents);
  return kvf_last_error();
}
