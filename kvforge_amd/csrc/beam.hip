// Beam search between two forward passes: which continuations of a request's beams live on, and what they own
// following them.
//
// Selection.  With logits l of a beam's row and the beam's running score S, candidate (beam, token) scores
//   S + (l - m) - log(sum_t exp(l_t - m)),   m = max_t l_t,
// and the `count` best of a request are wanted, best first, equal scores by the lower beam, then the lower token.
// Logits that are NaN or -inf are no candidates and weigh nothing, +inf counts as the largest finite number, and
// beams whose score is not finite are passed over unread.  Tokens that the caller rules out are no candidates either, but weigh.
//
//   1. `beam_pieces_kernel`: a workgroup takes a piece of a row, which stays in its registers (E logits a lane), so the row is
//      read once.  Maximum, sum of exponentials, and the piece's `count` best, sorted.  They are found by a bound: the 64 largest logits of a wave's
//      lanes, sorted, give a `count`-th and a (count / 4)-th; at least `count` logits reach the best of the four waves' former and
//      the least of their latter, and seldom many more.  What reaches the larger of the two goes to a list in LDS, where
//      every entry counts those ahead of it: its place.  (Logits equal to the bound are taken in the order of their tokens, no
//      more than `count` a wave, so the list holds whatever the logits are.)
//      512 rows of 128,256 (263 MB) take 47 us, 5.5 TB/s: as much as a kernel that only reads reaches on this card.
//   2. `beam_best_kernel`: a workgroup a request joins the sums of a row's pieces in 64 bits (candidates of different
//      beams may lie closer than 32 bits tell apart: their order is the sums' order), then picks among the pieces' best by a
//      bound and by counting again.  Where equal scores let too many entries reach the bound, the sorted lists are merged
//      instead, those of a wave side by side: of two sorted lists the larger of a[i] and b[count - 1 - i] are the best of both,
//      and log2(count) exchanges sort them again.
//   (One kernel, in which the workgroup of a request that is done last goes on with 2, saves 3 us of the host's time but takes
//   longer on the device, since results have to pass the XCDs' L2s and 2's registers are 1's too: 4 rows of 8,192 logits 13.4 us
//   against 10.3, 32 rows of 128,256 18.0 against 13.6, 512 rows 79 against 62, when it was tried.)
//
// Reordering: see `beam_reorder_kernel`.
#include <type_traits>

#include "common.h"

namespace {
constexpr int THREADS = 256, NWAVES = THREADS / KVF_WAVE;
constexpr int MAX_COUNT = 64;
constexpr float LARGEST = 3.402823466e38f;

// The order of finite numbers as unsigned integers; 0 stands below all of them ("no candidate").
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.f);       // (-0 equals 0)
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// exp(x) for x <= 0 (-inf too) to a few 2^-24, without the bias that a rounded log2(e) gives all terms of a sum.
__device__ __forceinline__ float exp_unbiased(float x) {
  constexpr float L = 1.44269504088896340736f;
  constexpr float L_LO = static_cast<float>(1.44269504088896340736 - static_cast<double>(L));
  static_assert(L_LO > 0.f, "-inf has to stay -inf");
  return __builtin_amdgcn_exp2f(fmaf(x, L_LO, x * L));
}

// The value of lane ^ O (O = 1 .. 63 of the forms below) without the LDS crossbar where it lies in the same 16 lanes: 1 and 2 are
// permutations of four lanes, 7 and 15 the mirrors of 8 and 16, and 4 = 7 ^ 3, 8 = 15 ^ 7.
template <int O> __device__ __forceinline__ uint32_t of_lane(uint32_t v) {
  auto dpp = [](uint32_t x, auto ctrl) { return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, true)); };
  if constexpr (O == 1) return dpp(v, std::integral_constant<int, 0xB1>{});
  else if constexpr (O == 2) return dpp(v, std::integral_constant<int, 0x4E>{});
  else if constexpr (O == 3) return dpp(v, std::integral_constant<int, 0x1B>{});
  else if constexpr (O == 7) return dpp(v, std::integral_constant<int, 0x141>{});
  else if constexpr (O == 15) return dpp(v, std::integral_constant<int, 0x140>{});
  else if constexpr (O == 4) return of_lane<3>(of_lane<7>(v));
  else if constexpr (O == 8) return of_lane<7>(of_lane<15>(v));
  else return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), O, KVF_WAVE));
}
template <int O> __device__ __forceinline__ unsigned long long of_lane(unsigned long long v) {
  return static_cast<unsigned long long>(of_lane<O>(static_cast<uint32_t>(v >> 32))) << 32 | of_lane<O>(static_cast<uint32_t>(v));
}
template <int O> __device__ __forceinline__ double of_lane(double v) {
  return __longlong_as_double(static_cast<long long>(of_lane<O>(static_cast<unsigned long long>(__double_as_longlong(v)))));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += of_lane<1>(v);
  v += of_lane<2>(v);
  v += of_lane<7>(v);       // the other four of 8 lanes
  v += of_lane<15>(v);      // the other eight of 16
  v += of_lane<16>(v);
  return v + of_lane<32>(v);
}
__device__ __forceinline__ float wave_most(float v) {
  auto of = [](float x, auto o) { return __uint_as_float(of_lane<decltype(o)::value>(__float_as_uint(x))); };
  v = fmaxf(v, of(v, std::integral_constant<int, 1>{}));
  v = fmaxf(v, of(v, std::integral_constant<int, 2>{}));
  v = fmaxf(v, of(v, std::integral_constant<int, 7>{}));
  v = fmaxf(v, of(v, std::integral_constant<int, 15>{}));
  v = fmaxf(v, of(v, std::integral_constant<int, 16>{}));
  return fmaxf(v, of(v, std::integral_constant<int, 32>{}));
}

// One exchange of a bitonic sort, the larger key to the lower lane: O with its lower bits set compares mirrored halves, a power of
// two the halves themselves.
template <int O> __device__ __forceinline__ void order_lanes(uint32_t& key, int lane) {
  const uint32_t other = of_lane<O>(key);
  const bool lower = (lane & ((O & (O - 1)) ? (O + 1) / 2 : O)) == 0;
  const uint32_t more = key > other ? key : other, less = key > other ? other : key;
  key = lower ? more : less;
}
// The `count`-th and the `few`-th largest of 64 lanes' keys: sorted, in about a hundred instructions (settling a threshold bit by
// bit takes four times as many).
__device__ __forceinline__ void kth_of_lanes(uint32_t key, int count, int few, uint32_t& kth, uint32_t& high) {
  const int lane = threadIdx.x % KVF_WAVE;
  order_lanes<1>(key, lane);
  order_lanes<3>(key, lane), order_lanes<1>(key, lane);
  order_lanes<7>(key, lane), order_lanes<2>(key, lane), order_lanes<1>(key, lane);
  order_lanes<15>(key, lane), order_lanes<4>(key, lane), order_lanes<2>(key, lane), order_lanes<1>(key, lane);
  order_lanes<31>(key, lane), order_lanes<8>(key, lane), order_lanes<4>(key, lane), order_lanes<2>(key, lane), order_lanes<1>(key, lane);
  order_lanes<63>(key, lane), order_lanes<16>(key, lane), order_lanes<8>(key, lane), order_lanes<4>(key, lane), order_lanes<2>(key, lane), order_lanes<1>(key, lane);
  kth = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), count - 1));
  high = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), few - 1));
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

__device__ __forceinline__ bool alive(float score) { return fabsf(score) <= LARGEST; }

// A wave's part of the list: what is strictly ahead of the bound lies in fewer than `count` of its lanes, equals are `count`
// at most; then zeros up to a whole step.
constexpr int LIST_STEP = 8;
__host__ __device__ __forceinline__ int list_room(int count, int e) { return ((count - 1) * e + count + 2 * LIST_STEP - 1) / LIST_STEP * LIST_STEP; }

struct PieceArgs {
  long stride;          // elements from one row of logits to the next
  int rows, vocab, count, pieces, piece;   // `piece`: elements of a piece, a multiple of THREADS * Chunk::N
  int n_ruled;          // tokens that are ruled out
};

// sums[row][piece] = (sum of exponentials, their reference), values/tokens[row][piece][count]: sorted, token -1 behind the last.
// RULED: the sum is made first, from the same logits in the same order, then the tokens in `ruled` leave the registers: a bit for each
// logit of the piece, set by whatever thread comes to the token (or-ing has no order).  4 rows of 8,192, 8 best: 8.6, 8.6, 9.0 us with 2, 43
// and 1,000 tokens, 8.2 without; 512 rows of 128,256, 16 best: 58.9, 59.1, 65.0, 52.0 without.
template <typename T, int E, bool RULED>
__global__ __launch_bounds__(THREADS) void beam_pieces_kernel(const T* __restrict__ logits, const float* __restrict__ scores,
                                                              double2* __restrict__ sums, float* __restrict__ values,
                                                              int* __restrict__ tokens, const int* __restrict__ ruled, PieceArgs a) {
  constexpr int N = Chunk<T>::N, CHUNKS = E / N;
  extern __shared__ __align__(16) unsigned long long list[];
  // list: (key, ~token) of what reaches the bound, a part for every wave
  __shared__ uint32_t bound_of[NWAVES], share_of[NWAVES];
  __shared__ float max_of[NWAVES];
  __shared__ double sum_of[NWAVES];
  __shared__ int n_of[NWAVES];
  const int tid = threadIdx.x, lane = tid % KVF_WAVE, wave = tid / KVF_WAVE;
  const int row = blockIdx.y, piece = blockIdx.x;
  if (!alive(scores[row])) return;       // the whole workgroup: such rows are passed over
  const size_t at = static_cast<size_t>(row) * a.pieces + piece;
  const T* x = logits + row * a.stride;
  // chunks lie on 16 bytes of memory: element e of the row is place e + skip of its first chunk's line
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const int lo = piece * a.piece - skip;        // the piece's first element (below 0 in front of the row)
  const int hi = min(lo + a.piece, a.vocab);
  float v[CHUNKS][N];
  if (lo >= 0 && lo + a.piece <= a.vocab) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) Chunk<T>::load(x + lo + (c * THREADS + tid) * N, v[c]);
  } else {
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
  }
  // NaN becomes -inf (the maximum is the other operand), +inf the largest finite number
  float top[CHUNKS], mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    top[c] = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[c][i] = fmaxf(v[c][i], -INFINITY);
      top[c] = fmaxf(top[c], v[c][i]);
    }
    mx = fmaxf(mx, top[c]);
  }
  if (__any(mx > LARGEST)) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      top[c] = fminf(top[c], LARGEST);
#pragma unroll
      for (int i = 0; i < N; ++i) v[c][i] = fminf(v[c][i], LARGEST);
    }
    mx = fminf(mx, LARGEST);
  }
  float m = -INFINITY;
  double s = 0.0;
  auto sum_up = [&] {
    if (m > -INFINITY) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float part = 0.f;             // of neighbours; the lane's sum is 64 bits wide
#pragma unroll
        for (int i = 0; i < N; ++i) part += exp_unbiased(v[c][i] - m);
        s += static_cast<double>(part);
      }
    }
    s = wave_sum64(s);
  };
  if constexpr (RULED) {
    __shared__ uint32_t out_bits[THREADS * E / 32];
    const float wmx = wave_most(mx);
    if (lane == 0) max_of[wave] = wmx;
    if (tid < THREADS * E / 32) out_bits[tid] = 0u;
    static_assert(E <= 32, "a word a thread at most");
    __syncthreads();
    for (int k = tid; k < a.n_ruled; k += THREADS) {
      const int token = ruled[k];
      if (token >= 0 && token >= lo && token < hi) atomicOr(&out_bits[(token - lo) / 32], 1u << ((token - lo) % 32));
    }
#pragma unroll
    for (int w = 0; w < NWAVES; ++w) m = fmaxf(m, max_of[w]);
    sum_up();
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int at0 = (c * THREADS + tid) * N;
      const uint32_t out = out_bits[at0 / 32] >> (at0 % 32);
#pragma unroll
      for (int i = 0; i < N; ++i) v[c][i] = out >> i & 1u ? -INFINITY : v[c][i];
    }
    mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      top[c] = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i) top[c] = fmaxf(top[c], v[c][i]);
      mx = fmaxf(mx, top[c]);
    }
  }
  const uint32_t lane_key = mx > -INFINITY ? order_key(mx) : 0u;
  uint32_t wave_bound, wave_share;
  kth_of_lanes(lane_key, a.count, (a.count + NWAVES - 1) / NWAVES, wave_bound, wave_share);
  const float wmx = RULED ? 0.f : wave_most(mx);
  if (lane == 0) {
    bound_of[wave] = wave_bound;
    share_of[wave] = wave_share;
    if (!RULED) max_of[wave] = wmx;
  }
  __syncthreads();
  // `count` logits reach every wave's own bound, and the least of the waves' shares
  uint32_t bound = share_of[0];
#pragma unroll
  for (int w = 1; w < NWAVES; ++w) bound = share_of[w] < bound ? share_of[w] : bound;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) {
    bound = bound_of[w] > bound ? bound_of[w] : bound;
    if (!RULED) m = fmaxf(m, max_of[w]);
  }
  // What is ahead of the bound, and what equals it in the order of the tokens.  Without a bound everything finite is taken.
  const unsigned long long below = (1ull << lane) - 1ull;
  const float least = bound ? key_value(bound) : -LARGEST;
  const int room = list_room(a.count, E);
  unsigned long long* mine = list + wave * room;
  int held = 0, ties = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (!__ballot(top[c] >= least)) continue;
    const int e = lo + (c * THREADS + tid) * N;
    unsigned long long same[N], equal = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      same[i] = __ballot(v[c][i] >= least);
      if (!same[i]) continue;
      const unsigned long long who = __ballot(v[c][i] > least);
      if (v[c][i] > least)
        mine[held + __popcll(who & below)] = static_cast<unsigned long long>(order_key(v[c][i])) << 32 | static_cast<uint32_t>(~(e + i));
      held += __popcll(who);
      same[i] &= ~who;
      equal |= same[i];
    }
    if (equal && ties < a.count) {
      int before = ties;            // equals of lower tokens
#pragma unroll
      for (int i = 0; i < N; ++i) {
        before += __popcll(same[i] & below);
        ties += __popcll(same[i]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!same[i]) continue;
        const bool is = same[i] >> lane & 1ull;
        const unsigned long long who = __ballot(is && before < a.count);
        if (is && before < a.count)
          mine[held + __popcll(who & below)] = static_cast<unsigned long long>(order_key(least)) << 32 | static_cast<uint32_t>(~(e + i));
        held += __popcll(who);
        before += is;
      }
    }
  }
  if (!RULED) sum_up();
  if (lane < LIST_STEP) mine[held + lane] = 0ull;       // the list is read in steps
  if (lane == 0) {
    sum_of[wave] = s;
    n_of[wave] = held;
  }
  __syncthreads();
  // Every entry counts those ahead of it: its place.  Four lanes an entry, each over the part of one wave.
  static_assert(NWAVES == 4, "a lane a part");
  float* out_v = values + at * a.count;
  int* out_t = tokens + at * a.count;
  int upto[NWAVES];
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) upto[w] = n_of[w] + (w ? upto[w - 1] : 0);
  const int n = upto[NWAVES - 1];
  const auto* other = reinterpret_cast<const ulonglong2*>(list + (tid % NWAVES) * room);
  const int others = n_of[tid % NWAVES];
  for (int i0 = 0; i0 < n; i0 += THREADS / NWAVES) {
    const int i = i0 + tid / NWAVES;
    unsigned long long entry = 0ull;
    if (i < n) entry = i < upto[0] ? list[i] : i < upto[1] ? list[room + i - upto[0]] : i < upto[2] ? list[2 * room + i - upto[1]] : list[3 * room + i - upto[2]];
    int place = 0;
    for (int k = 0; k < others; k += LIST_STEP) {
      ulonglong2 e[LIST_STEP / 2];
#pragma unroll
      for (int u = 0; u < LIST_STEP / 2; ++u) e[u] = other[k / 2 + u];
#pragma unroll
      for (int u = 0; u < LIST_STEP / 2; ++u) place += (e[u].x > entry) + (e[u].y > entry);
    }
    place += static_cast<int>(of_lane<1>(static_cast<uint32_t>(place)));
    place += static_cast<int>(of_lane<2>(static_cast<uint32_t>(place)));
    if (tid % NWAVES == 0 && i < n && place < a.count) {
      out_v[place] = key_value(static_cast<uint32_t>(entry >> 32));
      out_t[place] = static_cast<int>(~static_cast<uint32_t>(entry));
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
struct __align__(16) Entry {
  double score;
  unsigned long long tie;
};
constexpr unsigned long long NOBODY = ~0ull;
__device__ __forceinline__ bool ahead(const Entry& a, const Entry& b) {
  return a.score > b.score || (a.score == b.score && a.tie < b.tie);
}
template <int O> __device__ __forceinline__ Entry entry_of(const Entry& e) {
  return {of_lane<O>(e.score), of_lane<O>(e.tie)};
}

// The best L of two sorted lists of L that lie in groups of L lanes (L a power of two), sorted.
template <int O> __device__ __forceinline__ void exchange(Entry& e, int lane) {
  if constexpr (O > 0) {
    const Entry n = entry_of<O>(e);
    if (((lane & O) == 0) == ahead(n, e)) e = n;
    exchange<O / 2>(e, lane);
  }
}
template <int L> __device__ __forceinline__ Entry merge_lists(Entry mine, Entry other_reversed, int lane) {
  Entry e = ahead(mine, other_reversed) ? mine : other_reversed;
  exchange<L / 2>(e, lane);
  return e;
}
// The lists of a wave's groups of L lanes, O lanes apart and more within LANES, as one in every group.
template <int L, int O, int LANES = KVF_WAVE> __device__ __forceinline__ void merge_groups(Entry& e, int lane) {
  if constexpr (O < LANES) {
    e = merge_lists<L>(e, entry_of<O ^ (L - 1)>(e), lane);
    merge_groups<L, 2 * O, LANES>(e, lane);
  }
}

struct BestArgs {
  int rows, requests, count, pieces;
};
constexpr int BATCH = 64;       // rows of a request that are merged at a time
constexpr int FEW = 512;        // entries that are put in order by counting those ahead of each

constexpr int BEST_WAVES = 8, BEST_THREADS = BEST_WAVES * KVF_WAVE;

struct Survivors {
  Entry entry[FEW + 8];
  int token[FEW];
  uint32_t bound_of[BEST_WAVES], share_of[BEST_WAVES];
  int n;
};
template <int L> struct Merged {
  Entry entry[BEST_WAVES][L];
};

// (reference, S - log(sum)) of a row, in all lanes of the wave; (-inf, -inf) of one that has ended or has no candidate.
// `mine`: the sums of piece `lane`.
__device__ __forceinline__ double2 join_sums(const double2* p, double2 mine, float score, int pieces) {
  const int lane = threadIdx.x % KVF_WAVE;
  double m = -INFINITY, s = 0.0;
  if (alive(score)) {
    float most = static_cast<float>(mine.y);      // (a logit)
    for (int i = lane + KVF_WAVE; i < pieces; i += KVF_WAVE) most = fmaxf(most, static_cast<float>(p[i].y));
    m = wave_most(most);
    if (m > -INFINITY) {
      s = mine.x * exp(mine.y - m);
      for (int i = lane + KVF_WAVE; i < pieces; i += KVF_WAVE) s += p[i].x * exp(p[i].y - m);
    }
    s = wave_sum64(s);
  }
  return make_double2(m, s > 0.0 ? static_cast<double>(score) - log(s) : -INFINITY);
}
// What tells equal scores apart: see `Entry`.
__device__ __forceinline__ unsigned long long tie_of(int beam, float value, int place) {
  return static_cast<unsigned long long>(beam) << 48 | static_cast<unsigned long long>(~order_key(value)) << 16 | static_cast<unsigned long long>(place);
}
// The upper half of a score's order as an integer: scores in order have it in order (equal ones perhaps).
__device__ __forceinline__ uint32_t upper_key(double s) {
  const uint32_t b = static_cast<uint32_t>(static_cast<unsigned long long>(__double_as_longlong(s)) >> 32);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

// A wave's way through the entries of its rows (wave, wave + BEST_WAVES, ... of the request, `per_row` entries a lane each).  Lists
// are sorted, so lanes are turned against them from step to step: the best of a list do not all fall to the same lanes, and the
// bound, which goes by the lanes' best, is near.
struct Walk {
  int beam, part, turn;
  __device__ __forceinline__ int entry() const { return part * KVF_WAVE + ((threadIdx.x + turn) & (KVF_WAVE - 1)); }
  __device__ __forceinline__ void next(int per_row) {
    if (++part == per_row) part = 0, beam += BEST_WAVES;
    turn += 7;
  }
};
constexpr int SLOTS = 4;        // entries a lane has in its registers at a time

// All entries of a request's rows, a wave a row: the same bound as for a piece, by the upper halves of the scores, then every
// entry that reaches it counts those ahead.  False where more than FEW do (equal scores, mostly).
__device__ __forceinline__ bool best_by_counting(const float* scores, const double2* sums, const float* values, const int* tokens, int first,
                                                 int beams, int request, float* out_scores, int* out_beams, int* out_tokens,
                                                 const BestArgs& a, double2* row_of, Survivors& x) {
  const int tid = threadIdx.x, lane = tid % KVF_WAVE, wave = tid / KVF_WAVE;
  const int entries = a.pieces * a.count, per_row = (entries + KVF_WAVE - 1) / KVF_WAVE;
  if (beams > BATCH) return false;
  if (beams == 0) {
    if (tid < a.count) {
      const size_t to = static_cast<size_t>(request) * a.count + tid;
      out_scores[to] = -INFINITY;
      out_beams[to] = out_tokens[to] = -1;
    }
    return true;
  }
  const int slots = (beams + BEST_WAVES - 1 - wave) / BEST_WAVES * per_row;
  float value[SLOTS];
  int token[SLOTS];
  auto load = [&](Walk w) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const int e = w.entry();
      const bool there = w.beam < beams && e < entries;
      const size_t from = there ? static_cast<size_t>(first + w.beam) * entries + e : 0;
      const int read = tokens[from];          // (always: loads behind conditions go one by one)
      value[k] = values[from];
      token[k] = there ? read : -1;
      w.next(per_row);
    }
  };
  load({wave, 0, 0});
  for (int b = wave; b < beams; b += BEST_WAVES) {
    const int row = first + b;
    const float score = scores[row];
    const double2* p = sums + static_cast<size_t>(row) * a.pieces;
    const double2 mine = lane < a.pieces ? p[lane] : make_double2(0.0, -INFINITY);
    const double2 r = join_sums(p, mine, score, a.pieces);
    if (lane == 0) row_of[b] = r;
  }
  if (tid == 0) x.n = 0;
  // (row_of is this wave's own)
  double s[SLOTS];
  auto score_all = [&](Walk w) {
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const double2 r = row_of[min(w.beam, beams - 1)];
      s[k] = token[k] >= 0 && r.y > -INFINITY ? (static_cast<double>(value[k]) - r.x) + r.y : -INFINITY;
      w.next(per_row);
    }
  };
  uint32_t most = 0;
  Walk from{wave, 0, 0};
  for (int k0 = 0; k0 < slots; k0 += SLOTS) {
    Walk w = from;
    if (k0) load(w);
    score_all(w);
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const uint32_t key = s[k] > -INFINITY ? upper_key(s[k]) : 0u;
      most = key > most ? key : most;
      w.next(per_row);
    }
    from = w;
  }
  uint32_t kth, high;
  kth_of_lanes(most, a.count, (a.count + BEST_WAVES - 1) / BEST_WAVES, kth, high);
  if (lane == 0) {
    x.bound_of[wave] = kth;
    x.share_of[wave] = high;
  }
  __syncthreads();
  uint32_t bound = x.share_of[0];
#pragma unroll
  for (int w = 1; w < BEST_WAVES; ++w) bound = x.share_of[w] < bound ? x.share_of[w] : bound;
#pragma unroll
  for (int w = 0; w < BEST_WAVES; ++w) bound = x.bound_of[w] > bound ? x.bound_of[w] : bound;
  from = {wave, 0, 0};
  for (int k0 = 0; k0 < slots; k0 += SLOTS) {
    Walk w = from;
    if (slots > SLOTS) {
      load(w);
      score_all(w);
    }
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
      const bool takes = s[k] > -INFINITY && upper_key(s[k]) >= bound;
      const unsigned long long who = __ballot(takes);
      if (who) {
        int base = 0;
        if (lane == 0) base = atomicAdd(&x.n, static_cast<int>(__popcll(who)));
        const int to = __shfl(base, 0, KVF_WAVE) + __popcll(who & ((1ull << lane) - 1ull));
        if (takes && to < FEW) {
          x.entry[to] = {s[k], tie_of(w.beam, value[k], w.entry())};
          x.token[to] = token[k];
        }
      }
      w.next(per_row);
    }
    from = w;
  }
  __syncthreads();
  const int n = x.n;
  if (n > FEW) return false;
  // eight lanes an entry, each over every eighth
  constexpr int LANES = 8;
  for (int i0 = 0; i0 < n; i0 += BEST_THREADS / LANES) {
    const int i = i0 + tid / LANES;
    const Entry mine = x.entry[min(i, n - 1)];
    int place = 0;
    for (int j = tid % LANES; j < n; j += 2 * LANES) {
      const Entry one = x.entry[j], two = x.entry[j + LANES];
      place += ahead(one, mine) + (j + LANES < n && ahead(two, mine));
    }
    place += static_cast<int>(of_lane<1>(static_cast<uint32_t>(place)));
    place += static_cast<int>(of_lane<2>(static_cast<uint32_t>(place)));
    place += static_cast<int>(of_lane<7>(static_cast<uint32_t>(place)));
    if (tid % LANES == 0 && i < n && place < a.count) {
      const size_t to = static_cast<size_t>(request) * a.count + place;
      out_scores[to] = static_cast<float>(mine.score);
      out_beams[to] = static_cast<int>(mine.tie >> 48);
      out_tokens[to] = x.token[i];
    }
  }
  for (int i = n + tid; i < a.count; i += BEST_THREADS) {
    const size_t to = static_cast<size_t>(request) * a.count + i;
    out_scores[to] = -INFINITY;
    out_beams[to] = -1;
    out_tokens[to] = -1;
  }
  return true;
}

// The same for any number of entries: the sorted lists of all rows merged, those of a wave side by side.  L: `count` rounded up
// to a power of two.
template <int L>
__device__ __forceinline__ void best_by_merging(const float* scores, const double2* sums, const float* values, const int* tokens, int first,
                                                int beams, int request, float* out_scores, int* out_beams, int* out_tokens,
                                                const BestArgs& a, double2* row_of, Merged<L>& x) {
  constexpr int SIDE = KVF_WAVE / L;
  const int tid = threadIdx.x, lane = tid % KVF_WAVE, wave = tid / KVF_WAVE, group = lane / L, at = lane % L;
  Entry best{-INFINITY, NOBODY};
  for (int b0 = 0; b0 < beams; b0 += BATCH) {
    const int n = min(BATCH, beams - b0), lists = n * a.pieces;
    const size_t base = static_cast<size_t>(first + b0) * a.pieces;
    __syncthreads();
    for (int b = wave; b < n; b += BEST_WAVES) {
      const int row = first + b0 + b;
      const double2* p = sums + static_cast<size_t>(row) * a.pieces;
      const double2 r = join_sums(p, lane < a.pieces ? p[lane] : make_double2(0.0, -INFINITY), scores[row], a.pieces);
      if (lane == 0) row_of[b] = r;
    }
    __syncthreads();
    // `best` is sorted, so the other list is taken from its end
    const int i = L - 1 - at;
    for (int l = wave * SIDE + group; l - group < lists; l += BEST_WAVES * SIDE) {
      Entry e{-INFINITY, NOBODY};
      if (l < lists && i < a.count) {
        const int beam = l / a.pieces;
        const size_t from = (base + l) * a.count + i;
        const double2 r = row_of[beam];
        if (r.y > -INFINITY && tokens[from] >= 0) {
          e.score = (static_cast<double>(values[from]) - r.x) + r.y;
          e.tie = tie_of(b0 + beam, values[from], (l - beam * a.pieces) * a.count + i);
        }
      }
      best = merge_lists<L>(best, e, lane);
    }
  }
  merge_groups<L, L>(best, lane);
  if (lane < L) x.entry[wave][lane] = best;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < BEST_WAVES; ++w) best = merge_lists<L>(best, x.entry[w][L - 1 - at], lane);
  if (lane < a.count) {
    const bool there = best.tie != NOBODY;
    const int beam = static_cast<int>(best.tie >> 48);
    const size_t to = static_cast<size_t>(request) * a.count + lane;
    out_scores[to] = there ? static_cast<float>(best.score) : -INFINITY;
    out_beams[to] = there ? beam : -1;
    out_tokens[to] = there ? tokens[static_cast<size_t>(first + beam) * a.pieces * a.count + (best.tie & 0xffffull)] : -1;
  }
}

template <int L>
__global__ __launch_bounds__(BEST_THREADS) void beam_best_kernel(const float* scores, const int* __restrict__ cu_beams, const double2* sums,
                                                            const float* values, const int* tokens, float* out_scores, int* out_beams,
                                                            int* out_tokens, BestArgs a) {
  __shared__ union {
    Survivors few;
    Merged<L> merged;
  } x;
  __shared__ double2 row_of[BATCH];
  const int request = blockIdx.x;
  const int first = min(max(cu_beams[request], 0), a.rows);
  const int beams = min(max(cu_beams[request + 1], first), a.rows) - first;
  if (best_by_counting(scores, sums, values, tokens, first, beams, request, out_scores, out_beams, out_tokens, a, row_of, x.few)) return;
  __syncthreads();
  best_by_merging<L>(scores, sums, values, tokens, first, beams, request, out_scores, out_beams, out_tokens, a, row_of, x.merged);
}

template <typename T, int E>
int pieces_launch(const void* logits, const float* scores, double2* sums, float* values, int* tokens, const int* ruled, const PieceArgs& a,
                  hipStream_t stream) {
  const size_t lds = static_cast<size_t>(NWAVES) * list_room(a.count, E) * sizeof(unsigned long long);
  const dim3 grid(a.pieces, a.rows);
  const T* x = static_cast<const T*>(logits);
  if (a.n_ruled) beam_pieces_kernel<T, E, true><<<grid, THREADS, lds, stream>>>(x, scores, sums, values, tokens, ruled, a);
  else beam_pieces_kernel<T, E, false><<<grid, THREADS, lds, stream>>>(x, scores, sums, values, tokens, ruled, a);
  return kvf_last_error();
}
}  // namespace

// logits [rows][stride] of `vocab` (bf16: 0 fp32, 1 bf16); scores [rows]; cu_beams [requests + 1]; out_* [requests][count].
// Workspace: sums [rows][pieces][2] in 64 bits, values/tokens [rows][pieces][count].  piece: elements of a piece, 256 times 8,
// 16, or 32 for up to 32 candidates.  ruled [n_ruled]: tokens that are no candidates, in any order (others than the vocabulary's say
// nothing).
KVF_EXPORT int kvf_beam_select(int bf16, const void* logits, long stride, int rows, int vocab, const float* scores,
                               const int* cu_beams, int requests, int count, int pieces, int piece, void* sums,
                               float* values, int* tokens, float* out_scores, int* out_beams, int* out_tokens, const int* ruled,
                               int n_ruled, hipStream_t stream) {
  if (count < 1 || count > MAX_COUNT || n_ruled < 0 || rows < 0 || rows > 65535 || vocab < 1 || pieces < 1 || requests < 0 ||
      static_cast<long>(pieces) * count > 65536)
    return static_cast<int>(hipErrorInvalidValue);
  if (piece != THREADS * 8 && piece != THREADS * 16 && (piece != THREADS * 32 || count > 32)) return static_cast<int>(hipErrorInvalidValue);
  if (requests == 0) return 0;
  // a row may begin up to 15 bytes into its first chunk
  if (static_cast<long>(pieces) * piece < static_cast<long>(vocab) + (bf16 ? 7 : 3)) return static_cast<int>(hipErrorInvalidValue);
  auto* sum = static_cast<double2*>(sums);
  if (rows) {
    const PieceArgs a{stride, rows, vocab, count, pieces, piece, n_ruled};
#define KVF_PIECES(T) (piece == THREADS * 8    ? pieces_launch<T, 8>(logits, scores, sum, values, tokens, ruled, a, stream)   \
                       : piece == THREADS * 16 ? pieces_launch<T, 16>(logits, scores, sum, values, tokens, ruled, a, stream)  \
                                               : pieces_launch<T, 32>(logits, scores, sum, values, tokens, ruled, a, stream))
    const int rc = bf16 ? KVF_PIECES(bf16_t) : KVF_PIECES(float);
#undef KVF_PIECES
    if (rc) return rc;
  }
  const BestArgs b{rows, requests, count, pieces};
#define KVF_BEST(L) beam_best_kernel<L><<<requests, BEST_THREADS, 0, stream>>>(scores, cu_beams, sum, values, tokens, out_scores, out_beams, out_tokens, b)
  if (count <= 8) KVF_BEST(8);
  else if (count <= 16) KVF_BEST(16);
  else if (count <= 32) KVF_BEST(32);
  else KVF_BEST(64);
#undef KVF_BEST
  return kvf_last_error();
}

namespace {
constexpr int TILE_BYTES = THREADS * 16;
// Up to TILE_BYTES bytes of a tensor's row 0 from `base` on; rows are `stride` bytes apart and moved `unit` bytes at a time.
struct Tile {
  char* base;
  long stride;
  int bytes, unit;
};

// Where the rows of a request's beams come from and go to; row -1: nothing moves.  A lane a beam, so that two loads find out
// about all of them.
template <int W> struct Moves {
  int from[W], to[W];
  __device__ __forceinline__ void read(const int* __restrict__ slots, const int* __restrict__ parents, int beams, int rows) {
    const int lane = threadIdx.x % KVF_WAVE;
    const int p = lane < beams ? parents[lane] : -1, dst = lane < beams ? slots[lane] : -1;
    const bool named = p != lane && p >= 0 && p < beams;
    const int src = __shfl(dst, named ? p : lane, KVF_WAVE);
    const bool moves = named && dst >= 0 && dst < rows && src >= 0 && src < rows && src != dst;
#pragma unroll
    for (int b = 0; b < W; ++b) {
      from[b] = __builtin_amdgcn_readlane(moves ? src : -1, b);
      to[b] = __builtin_amdgcn_readlane(moves ? dst : -1, b);
    }
  }
};

// Bytes of device memory, by the type that they are moved as: vectors of the language (arrays of HIP's own go through LDS) behind
// pointers known to be global (one read from a table may point anywhere, and its loads wait on the LDS counter too).
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));
typedef uint32_t Word2 __attribute__((ext_vector_type(2)));
template <typename Unit> __device__ __forceinline__ Unit get(const char* base, long at) {
  return *(const __attribute__((address_space(1))) Unit*)(base + at);
}
template <typename Unit> __device__ __forceinline__ void put(char* base, long at, Unit v) {
  *(__attribute__((address_space(1))) Unit*)(base + at) = v;
}

// All loads have arrived, and the compiler knows it: otherwise it waits again ahead of every store, and with it for the stores
// before (eight requests of four beams, 1 MB rows of eight tensors: 101 us, and 37 so).
__device__ __forceinline__ void loads_arrived() {
  __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt 0, the other counters as they are
  asm volatile("" ::: "memory");
}

// Tiles of all rows of a request: a lane's bytes of every row that moves are in its registers before it writes any of them, and
// no other lane touches them, so rows may change places in any way (swaps and rings too) without memory beside them.
// What bounds it: bytes, each row that moves read and written once.  32 requests of 8 beams, 64 tensors of 32 KB rows: 349 MB in
// 74 us from memory, 4.7 TB/s, as much as a plain copy of that size; 8 of 4 beams, 8 tensors of 1 MB rows: 160 MB in 37 us.
// More bytes a lane do not help (tiles a workgroup U = 1, 2, 4, 8 for four beams: 43.8, 43.9, 46.2, 47.8 us): waves do.
//
// U tiles, a unit at a time; WHOLE: all of them are.  Units below 16 bytes lie THREADS apart, so that a lane has as many of them
// in flight as registers for 16 bytes hold (tensors of 4-byte units: 12 us with one at a time, 15 requests of 13 beams).
template <typename Unit, int W, int U, bool WHOLE> __device__ __forceinline__ void move_tiles(const Tile (&t)[U], const Moves<W>& m) {
  constexpr int SIZE = sizeof(Unit), PASSES = TILE_BYTES / (THREADS * SIZE), PER = PASSES < 4 ? PASSES : 4;
#pragma unroll 1
  for (int pass = 0; pass < PASSES; pass += PER) {
    Unit v[W][U][PER];
    auto place = [&](int p) { return ((pass + p) * THREADS + static_cast<int>(threadIdx.x)) * SIZE; };
#pragma unroll
    for (int b = 0; b < W; ++b)
      if (m.to[b] >= 0)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int p = 0; p < PER; ++p) {
            const int at = WHOLE ? place(p) : max(min(place(p), t[u].bytes - SIZE), 0);
            v[b][u][p] = get<Unit>(t[u].base + m.from[b] * t[u].stride, at);
          }
    loads_arrived();
#pragma unroll
    for (int b = 0; b < W; ++b)
      if (m.to[b] >= 0)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int p = 0; p < PER; ++p)
            if (WHOLE || place(p) < t[u].bytes) put(t[u].base + m.to[b] * t[u].stride, place(p), v[b][u][p]);
  }
}

template <int W, int U>
__global__ __launch_bounds__(THREADS) void beam_reorder_kernel(const Tile* __restrict__ tiles, int n_tiles, int rows, int beams,
                                                               const int* __restrict__ slots, const int* __restrict__ parents) {
  Tile t[U];
  bool whole = true;
  int unit = 16;                // that all of them can be moved by
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = blockIdx.x * U + u;
    t[u] = tiles[min(i, n_tiles - 1)];
    unit = min(unit, t[u].unit);
    if (i >= n_tiles) t[u].bytes = 0;
    whole &= t[u].bytes == TILE_BYTES;
  }
  Moves<W> m;
  m.read(slots + static_cast<size_t>(blockIdx.y) * beams, parents + static_cast<size_t>(blockIdx.y) * beams, beams, rows);
  if (unit == 16) {
    if (whole) move_tiles<Word4, W, U, true>(t, m);
    else move_tiles<Word4, W, U, false>(t, m);
  } else if (unit == 8) {
    move_tiles<Word2, W, U, false>(t, m);
  } else if (unit == 4) {
    move_tiles<uint32_t, W, U, false>(t, m);
  } else {
    move_tiles<uint16_t, W, U, false>(t, m);
  }
}

template <int W, int U>
void reorder_launch(const Tile* tiles, int n_tiles, int rows, int requests, int beams, const int* slots, const int* parents, hipStream_t stream) {
  beam_reorder_kernel<W, U><<<dim3((n_tiles + U - 1) / U, requests), THREADS, 0, stream>>>(tiles, n_tiles, rows, beams, slots, parents);
}
}  // namespace

KVF_EXPORT int kvf_beam_tile_bytes() { return TILE_BYTES; }

// tiles: Tile (address, bytes from row to row, bytes of the tile | unit << 32: three 64-bit numbers) each; slots, parents
// [requests][beams].
KVF_EXPORT int kvf_beam_reorder(const void* tiles, int n_tiles, int rows, int requests, int beams, const int* slots, const int* parents,
                                hipStream_t stream) {
  static_assert(sizeof(Tile) == 24, "as the table is written");
  if (beams < 1 || beams > 32 || requests < 0 || requests > 65535 || n_tiles < 0 || rows < 0) return static_cast<int>(hipErrorInvalidValue);
  if (requests == 0 || n_tiles == 0 || beams == 1) return 0;
  const auto* t = static_cast<const Tile*>(tiles);
  if (beams <= 4) reorder_launch<4, 2>(t, n_tiles, rows, requests, beams, slots, parents, stream);
  else if (beams <= 8) reorder_launch<8, 2>(t, n_tiles, rows, requests, beams, slots, parents, stream);
  else if (beams <= 16) reorder_launch<16, 2>(t, n_tiles, rows, requests, beams, slots, parents, stream);
  else reorder_launch<32, 1>(t, n_tiles, rows, requests, beams, slots, parents, stream);
  return kvf_last_error();
}
