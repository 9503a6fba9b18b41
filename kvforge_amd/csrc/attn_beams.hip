// Attention of one token per sequence over the paged cache where sequences come in groups whose first keys lie in the same
// pages (the beams of a request behind its prompt): the keys that a group shares are read once for all its rows.
//
//   out = softmax(scale * q K^T) V per head, over the keys [0, ctx) of the sequence; sinks: one more term exp(sink_h) in the
//   denominator.  A sequence without keys gets zeros.
//
// A workgroup of four waves takes a cut of a range of keys for one kv head and up to 16 * RT rows: of the shared keys, rows are
// (sequence of the group, head that shares the kv head); of a sequence's own keys, the heads alone.  Every cut leaves its
// (reference, sum, accumulator) in the workspace, and `attn_beams_join_kernel` joins the cuts of a row.
//
// Blocks of 32 keys go round the waves.  For lane l, g = l / 16, r = l % 16:
//   S^T (keys x rows) = K Q^T in two tiles t of 16 keys; tile row i is key 8 (i / 4) + 4 t + i % 4, so that a lane ends up with
//     the scores of the eight neighbouring keys 8 g .. 8 g + 7 of row r;
//   O^T (d x rows) += V^T P^T: V pages hold an element's keys side by side, so a lane's eight keys of one element are one load,
//     and its probabilities are the other operand as they stand (bf16: rounded once; fp32: v_mfma_f32_16x16x4_f32 takes them
//     key by key).
// Fragments come from the pages in this order, nothing is staged.  Lanes without a valid page read page 0 and are masked.
//
// A row's reference (what is subtracted in the exponent) is raised only when a score passes it by LAZY (in log2 units); scores,
// sums and accumulators are fp32.
#include "common.h"

namespace {
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
constexpr int WAVES = 4, THREADS = WAVES * KVF_WAVE;
constexpr int BLOCK = 32;              // keys a wave takes at a time
constexpr float LAZY = 8.f;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  int H, KV, d, bs, nb, width, q_stride, o_stride, n_seqs, n_groups;
  int blocks;          // row blocks of a group that have a workgroup of their own
  int cs, co;          // cuts of the shared keys and of a sequence's own
  float scale2;        // scale * log2(e)
  unsigned bs_magic;   // floor(2^32 / bs) + 1: key / bs == mulhi(key, bs_magic) while key * bs < 2^32
};

__device__ __forceinline__ int page_of(int key, const Args& a) { return static_cast<int>(__umulhi(static_cast<unsigned>(key), a.bs_magic)); }

// What differs between the element types: fragments of K (two tiles of a block), of V (16 elements by 32 keys), of Q.
template <typename T> struct Frag;
template <> struct Frag<bf16_t> {
  static constexpr int SLICE = 32;     // elements of d that one K or Q fragment spans over the lane groups
  typedef bf16x8 Part;                 // a lane's part of it
  struct Keys { bf16x8 v; };           // eight keys of one element
  static __device__ __forceinline__ Part zero() { return __builtin_bit_cast(Part, uint4{0, 0, 0, 0}); }
  static __device__ __forceinline__ Part load(const bf16_t* p) { return __builtin_bit_cast(Part, *reinterpret_cast<const uint4*>(p)); }
  static __device__ __forceinline__ f32x4 scores(Part k, Part q, f32x4 s) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q, s, 0, 0, 0); }
  static __device__ __forceinline__ Keys load_keys(const bf16_t* p) { return {load(p)}; }
  static __device__ __forceinline__ void set(Keys& k, int i, bf16_t v) { k.v[i] = __builtin_bit_cast(__bf16, v.bits); }
  static __device__ __forceinline__ void clear(Keys& k, unsigned keep) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k.v[i] = keep >> i & 1u ? k.v[i] : static_cast<__bf16>(0.f);
  }
  struct Probs { bf16x8 v; };
  static __device__ __forceinline__ Probs probs(const f32x4 (&p)[2]) {
    Probs o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = static_cast<__bf16>(p[i / 4][i % 4]);
    return o;
  }
  static __device__ __forceinline__ f32x4 values(const Keys& k, const Probs& p, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, p.v, acc, 0, 0, 0); }
};
template <> struct Frag<float> {
  static constexpr int SLICE = 16;
  typedef f32x4 Part;
  struct Keys { f32x4 v[2]; };
  static __device__ __forceinline__ Part zero() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ Part load(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
  static __device__ __forceinline__ f32x4 scores(Part k, Part q, f32x4 s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i], q[i], s, 0, 0, 0);
    return s;
  }
  static __device__ __forceinline__ Keys load_keys(const float* p) { return {{load(p), load(p + 4)}}; }
  static __device__ __forceinline__ void set(Keys& k, int i, float v) { k.v[i / 4][i % 4] = v; }
  static __device__ __forceinline__ void clear(Keys& k, unsigned keep) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k.v[i / 4][i % 4] = keep >> i & 1u ? k.v[i / 4][i % 4] : 0.f;
  }
  struct Probs { f32x4 v[2]; };
  static __device__ __forceinline__ Probs probs(const f32x4 (&p)[2]) { return {{p[0], p[1]}}; }
  static __device__ __forceinline__ f32x4 values(const Keys& k, const Probs& p, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k.v[i / 4][i % 4], p.v[i / 4][i % 4], acc, 0, 0, 0);
    return acc;
  }
};

template <typename T> struct Tensors {
  const T *q, *k, *v;
  const int *table, *cu_groups, *shared_lens, *ctx_lens;
  float* acc;
  float2* ml;
};

// The keys that the sequences [first, first + n) share: no more than the shortest of them that has any.  `holder`: the first
// that has any, whose pages they are read from.
__device__ __forceinline__ int shared_keys(int group, int first, int n, const int* shared_lens, const int* ctx_lens, int most, int& holder) {
  int least = most, who = n - 1;
  for (int i = threadIdx.x % KVF_WAVE; i < n; i += KVF_WAVE) {
    const int c = ctx_lens[first + i];
    if (c > 0) {
      least = min(least, c);
      who = min(who, i);
    }
  }
#pragma unroll
  for (int o = KVF_WAVE / 2; o > 0; o >>= 1) {
    least = min(least, __shfl_xor(least, o, KVF_WAVE));
    who = min(who, __shfl_xor(who, o, KVF_WAVE));
  }
  holder = first + who;
  return max(0, min(least, shared_lens[group]));
}

// Rows [row0, row0 + 16 RT) of `rows` (sequence first + row / G, head row % G of kv head `kvh`), keys [lo, hi) of the pages in
// `table`; results go to cut `cut`.  DT: tiles of 16 elements of d (at least d / 16).
template <typename T, int DT, int RT, bool ALIGNED>
__device__ void attend(const Tensors<T>& t, const Args& a, const int* __restrict__ table, int first, int rows, int row0, int kvh,
                       int lo, int hi, int cut, f32x4* lds_acc, float2* lds_ml) {
  typedef Frag<T> F;
  constexpr int SLICES = DT * 16 / F::SLICE, LANE_D = F::SLICE / 4;
  const int lane = threadIdx.x % KVF_WAVE, wave = threadIdx.x / KVF_WAVE, g = lane / 16, r = lane % 16;
  const int G = a.H / a.KV, d = a.d, tiles = d / 16;
  typename F::Part q[RT][SLICES];
  bool live[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = row0 + rt * 16 + r;
    const int seq = first + min(row, rows - 1) / G;
    live[rt] = row < rows && t.ctx_lens[seq] > 0;
    const T* from = t.q + static_cast<long>(seq) * a.q_stride + (kvh * G + min(row, rows - 1) % G) * d;
#pragma unroll
    for (int c = 0; c < SLICES; ++c) {
      const int e = c * F::SLICE + g * LANE_D;
      q[rt][c] = e < d ? F::load(from + e) : F::zero();
    }
  }
  f32x4 acc[RT][DT];
  float m[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const long page_elems = static_cast<long>(a.KV) * a.bs * d;
  const T* kp = t.k + static_cast<long>(kvh) * a.bs * d;
  const T* vp = t.v + static_cast<long>(kvh) * a.bs * d;
  // page numbers of the eight keys from `key` on (ALIGNED: one page), 0 and a cleared bit where there is none
  auto lookup = [&](int key, bool& ok) {
    const int p = key >= lo - 7 && key < hi ? table[page_of(key, a)] : -1;
    ok = p >= 0 && p < a.nb;
    return ok ? p : 0;
  };
  for (int kb = (lo & ~7) + wave * BLOCK; kb < hi; kb += WAVES * BLOCK) {
    typename F::Part kf[2][SLICES];
    typename F::Keys vf[DT];
    unsigned keep = 0;                // which of the lane's keys 8 g .. 8 g + 7 count
    if constexpr (ALIGNED) {
      bool ok_k, ok_v;
      const int key_k = kb + 8 * (r / 4), key_v = kb + 8 * g;
      const int pk = lookup(key_k, ok_k), pv = lookup(key_v, ok_v);
      const int off_k = ok_k ? key_k - page_of(key_k, a) * a.bs : 0, off_v = ok_v ? key_v - page_of(key_v, a) * a.bs : 0;
      const T* k0 = kp + pk * page_elems + static_cast<long>(off_k + r % 4) * d;
      const T* v0 = vp + pv * page_elems + off_v + r * a.bs;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int c = 0; c < SLICES; ++c) {
          const int e = c * F::SLICE + g * LANE_D;
          kf[tt][c] = e < d ? F::load(k0 + tt * 4 * d + e) : F::zero();
        }
#pragma unroll
      for (int j = 0; j < DT; ++j)
        if (j < tiles) vf[j] = F::load_keys(v0 + static_cast<long>(j) * 16 * a.bs);
      const int from = max(lo - key_v, 0), to = min(hi - key_v, 8);
      keep = ok_v && to > from ? (0xffu >> (8 - to)) & (0xffu << from) : 0u;
    } else {
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const int key = kb + 8 * (r / 4) + 4 * tt + r % 4;
        bool ok = false;
        int p = 0, off = 0;
        if (key >= lo && key < hi) {
          p = table[key / a.bs];
          ok = p >= 0 && p < a.nb;
          off = key % a.bs;
        }
        const T* k0 = kp + (ok ? p : 0) * page_elems + static_cast<long>(ok ? off : 0) * d;
#pragma unroll
        for (int c = 0; c < SLICES; ++c) {
          const int e = c * F::SLICE + g * LANE_D;
          kf[tt][c] = e < d ? F::load(k0 + e) : F::zero();
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = kb + 8 * g + i;
        bool ok = false;
        int p = 0, off = 0;
        if (key >= lo && key < hi) {
          p = table[key / a.bs];
          ok = p >= 0 && p < a.nb;
          off = key % a.bs;
        }
        keep |= ok ? 1u << i : 0u;
        const T* v0 = vp + (ok ? p : 0) * page_elems + (ok ? off : 0) + r * a.bs;
#pragma unroll
        for (int j = 0; j < DT; ++j)
          if (j < tiles) F::set(vf[j], i, v0[static_cast<long>(j) * 16 * a.bs]);
      }
    }
    const bool whole = __all(keep == 0xffu);
    if (!whole)
#pragma unroll
      for (int j = 0; j < DT; ++j)
        if (j < tiles) F::clear(vf[j], keep);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      f32x4 s[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        s[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < SLICES; ++c) s[tt] = F::scores(kf[tt][c], q[rt][c], s[tt]);
        s[tt] *= a.scale2;
        if (!whole)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[tt][i] = keep >> (4 * tt + i) & 1u ? s[tt][i] : -INFINITY;
      }
      float most = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) most = fmaxf(most, s[i / 4][i % 4]);
      if (__any(most > m[rt] + LAZY)) {
        most = fmaxf(most, __shfl_xor(most, 16, KVF_WAVE));
        most = fmaxf(most, __shfl_xor(most, 32, KVF_WAVE));
        const float raised = fmaxf(m[rt], most);
        const float by = raised > -INFINITY ? __builtin_amdgcn_exp2f(m[rt] - raised) : 1.f;
        m[rt] = raised;
        sum[rt] *= by;
#pragma unroll
        for (int j = 0; j < DT; ++j) acc[rt][j] *= by;
      }
      const float ref = m[rt] > -INFINITY ? m[rt] : 0.f;
      f32x4 p[2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i / 4][i % 4] = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - ref);
        sum[rt] += p[i / 4][i % 4];
      }
      const typename F::Probs pf = F::probs(p);
#pragma unroll
      for (int j = 0; j < DT; ++j)
        if (j < tiles) acc[rt][j] = F::values(vf[j], pf, acc[rt][j]);
    }
  }
  // the waves' results, one tile of rows at a time
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float l = sum[rt];
    l += __shfl_xor(l, 16, KVF_WAVE);
    l += __shfl_xor(l, 32, KVF_WAVE);
    __syncthreads();
    if (g == 0) lds_ml[wave * 16 + r] = make_float2(m[rt], l);
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_ml[w * 16 + r].x);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 o = lds_ml[w * 16 + r];
      total += o.x > -INFINITY || o.y != o.y ? o.y * __builtin_amdgcn_exp2f(o.x - top) : 0.f;     // (NaN stays NaN)
    }
    const float by = m[rt] > -INFINITY ? __builtin_amdgcn_exp2f(m[rt] - top) : 0.f;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      acc[rt][j] *= by;
      if (wave > 0 && j < tiles) lds_acc[((wave - 1) * DT + j) * KVF_WAVE + lane] = acc[rt][j];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int j = 0; j < DT; ++j)
        if (j < tiles) {
          f32x4 o = acc[rt][j];
#pragma unroll
          for (int w = 0; w < WAVES - 1; ++w) o += lds_acc[(w * DT + j) * KVF_WAVE + lane];
          acc[rt][j] = o;
        }
      const int row = row0 + rt * 16 + r;
      if (row < rows) {
        const int seq = first + row / G, h = kvh * G + row % G;
        const long at = (static_cast<long>(seq) * a.H + h) * (a.cs + a.co) + cut;
        const bool any = live[rt] && (total > 0.f || total != total);
        if (g == 0) t.ml[at] = any ? make_float2(top > -INFINITY ? top : 0.f, total) : make_float2(-INFINITY, 0.f);
        if (any)
#pragma unroll
          for (int j = 0; j < DT; ++j)
            if (j < tiles) *reinterpret_cast<f32x4*>(t.acc + at * d + j * 16 + g * 4) = acc[rt][j];
      }
    }
  }
}

// Cut `c` of `n` of the keys [lo, hi), in whole rounds of the waves.
__device__ __forceinline__ void cut_of(int& lo, int& hi, int c, int n) {
  const int first = lo & ~7, round = WAVES * BLOCK;
  const int per = ((hi - first + n - 1) / n + round - 1) / round * round;
  const int from = first + min(c * per, hi - first), to = min(from + per, hi);
  lo = max(lo, from);
  hi = to;
}

template <typename T, int DT, int RT, bool ALIGNED>
__global__ __launch_bounds__(THREADS) void attn_beams_kernel(Tensors<T> t, Args a) {
  __shared__ f32x4 lds_acc[(WAVES - 1) * DT * KVF_WAVE];
  __shared__ float2 lds_ml[WAVES * 16];
  const int shared_items = a.n_groups * a.cs * a.blocks * a.KV;
  const int G = a.H / a.KV, most = a.width * a.bs, lane = threadIdx.x % KVF_WAVE;
  int item = blockIdx.x;
  if (item < shared_items) {
    const int kvh = item % a.KV, block = item / a.KV % a.blocks, cut = item / a.KV / a.blocks % a.cs, group = item / a.KV / a.blocks / a.cs;
    const int first = min(max(t.cu_groups[group], 0), a.n_seqs), n = min(max(t.cu_groups[group + 1], first), a.n_seqs) - first;
    if (n == 0) return;
    int holder, lo = 0, hi = shared_keys(group, first, n, t.shared_lens, t.ctx_lens, most, holder);
    cut_of(lo, hi, cut, a.cs);
    for (int row0 = block * 16 * RT; row0 < n * G; row0 += a.blocks * 16 * RT)
      attend<T, DT, RT, ALIGNED>(t, a, t.table + static_cast<long>(holder) * a.width, first, n * G, row0, kvh, lo, hi, cut, lds_acc, lds_ml);
  } else {
    item -= shared_items;
    const int kvh = item % a.KV, cut = item / a.KV % a.co, seq = item / a.KV / a.co;
    // the group that the sequence is in
    int lo = 0;
    bool grouped = false;
    for (int g0 = 0; g0 < a.n_groups; g0 += KVF_WAVE) {
      const int g = min(g0 + lane, a.n_groups - 1);
      const unsigned long long here = __ballot(t.cu_groups[g] <= seq && seq < t.cu_groups[g + 1]);
      if (here) {
        const int group = min(g0 + __ffsll(static_cast<long long>(here)) - 1, a.n_groups - 1);
        const int first = max(t.cu_groups[group], 0);
        int holder;
        lo = a.cs ? shared_keys(group, first, min(t.cu_groups[group + 1], a.n_seqs) - first, t.shared_lens, t.ctx_lens, most, holder) : 0;
        grouped = true;
        break;
      }
    }
    if (!grouped && cut == 0)       // nobody else tells of its shared keys
      for (int i = threadIdx.x; i < G * a.cs; i += THREADS)
        t.ml[(static_cast<long>(seq) * a.H + kvh * G + i / a.cs) * (a.cs + a.co) + i % a.cs] = make_float2(-INFINITY, 0.f);
    int hi = max(lo, min(t.ctx_lens[seq], most));
    cut_of(lo, hi, cut, a.co);
    for (int row0 = 0; row0 < G; row0 += 16 * RT)
      attend<T, DT, RT, ALIGNED>(t, a, t.table + static_cast<long>(seq) * a.width, seq, G, row0, kvh, lo, hi, a.cs + cut, lds_acc, lds_ml);
  }
}

// A wave a row: the cuts' sums and accumulators at the largest of their references.  Lanes: four elements each, of up to four cuts
// side by side.
template <typename T>
__global__ __launch_bounds__(THREADS) void attn_beams_join_kernel(const float* __restrict__ acc, const float2* __restrict__ ml,
                                                                  T* __restrict__ out, const float* __restrict__ sinks, Args a) {
  const int lane = threadIdx.x % KVF_WAVE, cuts = a.cs + a.co;
  const long row = static_cast<long>(blockIdx.x) * WAVES + threadIdx.x / KVF_WAVE;
  if (row >= static_cast<long>(a.n_seqs) * a.H) return;
  const int h = static_cast<int>(row % a.H);
  const float2* mine = ml + row * cuts;
  float top = -INFINITY;
  for (int c = lane; c < cuts; c += KVF_WAVE) top = fmaxf(top, mine[c].x);
  top = wave_max(top);
  const bool any = top > -INFINITY;
  if (sinks != nullptr) top = fmaxf(top, sinks[h] * LOG2E);
  float total = 0.f;
  for (int c = lane; c < cuts; c += KVF_WAVE)
    if (mine[c].x > -INFINITY) total += mine[c].y * __builtin_amdgcn_exp2f(mine[c].x - top);
  total = wave_sum(total);
  if (sinks != nullptr) total += __builtin_amdgcn_exp2f(sinks[h] * LOG2E - top);
  const int quads = a.d / 4, side = quads > 32 ? 1 : quads > 16 ? 2 : 4;
  const int sub = lane / (KVF_WAVE / side), at = lane % (KVF_WAVE / side);
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  if (at < quads)
    for (int c = sub; c < cuts; c += side) {
      const float2 x = mine[c];
      if (x.x > -INFINITY) o += *reinterpret_cast<const f32x4*>(acc + (row * cuts + c) * a.d + at * 4) * __builtin_amdgcn_exp2f(x.x - top);
    }
  for (int s = KVF_WAVE / side; s < KVF_WAVE; s *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], s, KVF_WAVE);
  if (sub == 0 && at < quads) {
    T* to = out + row / a.H * a.o_stride + static_cast<long>(h) * a.d + at * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) Elem<T>::store(to + i, any ? o[i] / total : 0.f);
  }
}

// Heads up to so many elements have room in the registers for two tiles of rows a wave.
constexpr int TWO_TILES = 128;
int row_tiles_of(int d, int bs, int rows) { return rows > 16 && d <= TWO_TILES && bs % 8 == 0 ? 2 : 1; }

template <typename T, int DT, bool ALIGNED>
int launch_rows(const Tensors<T>& t, const Args& a, int row_tiles, hipStream_t stream) {
  const long items = (static_cast<long>(a.n_groups) * a.cs * a.blocks + static_cast<long>(a.n_seqs) * a.co) * a.KV;
  if (items > 0x7fffffffL) return static_cast<int>(hipErrorInvalidValue);
  const dim3 grid(static_cast<unsigned>(items));
  if constexpr (ALIGNED && DT <= TWO_TILES / 16) {
    if (row_tiles == 2) {
      attn_beams_kernel<T, DT, 2, ALIGNED><<<grid, THREADS, 0, stream>>>(t, a);
      return kvf_last_error();
    }
  }
  attn_beams_kernel<T, DT, 1, ALIGNED><<<grid, THREADS, 0, stream>>>(t, a);
  return kvf_last_error();
}
template <typename T, bool ALIGNED>
int launch_dims(const Tensors<T>& t, const Args& a, int row_tiles, hipStream_t stream) {
  if (a.d <= 32) return launch_rows<T, 2, ALIGNED>(t, a, row_tiles, stream);
  if (a.d <= 64) return launch_rows<T, 4, ALIGNED>(t, a, row_tiles, stream);
  if (a.d <= 96) return launch_rows<T, 6, ALIGNED>(t, a, row_tiles, stream);
  if (a.d <= 128) return launch_rows<T, 8, ALIGNED>(t, a, row_tiles, stream);
  return launch_rows<T, 16, ALIGNED>(t, a, row_tiles, stream);
}
template <typename T>
int run(const void* q, const void* k, const void* v, const int* table, const int* cu_groups, const int* shared_lens, const int* ctx_lens,
        void* out, float* acc, void* ml, const float* sinks, const Args& a, int row_tiles, hipStream_t stream) {
  const Tensors<T> t{static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), table, cu_groups, shared_lens, ctx_lens,
                     acc, static_cast<float2*>(ml)};
  const int rc = a.bs % 8 == 0 ? launch_dims<T, true>(t, a, row_tiles, stream) : launch_dims<T, false>(t, a, row_tiles, stream);
  if (rc) return rc;
  const long rows = static_cast<long>(a.n_seqs) * a.H;
  attn_beams_join_kernel<T><<<static_cast<unsigned>((rows + WAVES - 1) / WAVES), THREADS, 0, stream>>>(acc, static_cast<const float2*>(ml), static_cast<T*>(out), sinks, a);
  return kvf_last_error();
}
}  // namespace

// Tiles of 16 rows that a workgroup takes where a group has `rows` rows a kv head.
KVF_EXPORT int kvf_attn_beams_row_tiles(int d, int bs, int rows) { return row_tiles_of(d, bs, rows); }

// q [n_seqs] rows of H heads; pages k [nb, KV, bs, d], v [nb, KV, d, bs]; table [n_seqs, width]; cu_groups [n_groups + 1];
// shared_lens [n_groups]; ctx_lens [n_seqs].  Workspace: acc [n_seqs, H, cs + co, d], ml [n_seqs, H, cs + co, 2].
KVF_EXPORT int kvf_attn_beams(int bf16, const void* q, const void* k, const void* v, const int* table, const int* cu_groups,
                              const int* shared_lens, const int* ctx_lens, void* out, float* acc, void* ml, const float* sinks, int H,
                              int KV, int d, int bs, int nb, int width, int q_stride, int o_stride, int n_seqs, int n_groups, int widest,
                              int cs, int co, float scale, hipStream_t stream) {
  if (KV < 1 || H < KV || H % KV || d < 16 || d > 256 || d % 16 || bs < 1 || nb < 1 || width < 0 || n_seqs < 0 || n_groups < 0 ||
      widest < 1 || cs < 0 || co < 1 || cs > 64 || co > 64 || (n_groups == 0 && cs))
    return static_cast<int>(hipErrorInvalidValue);
  if (static_cast<long>(width) * bs >= (1L << 31) - 1024 || static_cast<long>(width) * bs * bs >= (1L << 32)) return static_cast<int>(hipErrorInvalidValue);
  if (n_seqs == 0) return 0;
  const long rows = static_cast<long>(widest) * (H / KV);
  if (rows > 1 << 20) return static_cast<int>(hipErrorInvalidValue);
  const int row_tiles = row_tiles_of(d, bs, static_cast<int>(rows)), blocks = static_cast<int>((rows + 16 * row_tiles - 1) / (16 * row_tiles));
  const Args a{H, KV, d, bs, nb, width, q_stride, o_stride, n_seqs, n_groups, blocks, cs, co, scale * LOG2E,
               bs > 1 ? static_cast<unsigned>((1ull << 32) / bs) + 1u : 0u};
  return bf16 ? run<bf16_t>(q, k, v, table, cu_groups, shared_lens, ctx_lens, out, acc, ml, sinks, a, row_tiles, stream)
              : run<float>(q, k, v, table, cu_groups, shared_lens, ctx_lens, out, acc, ml, sinks, a, row_tiles, stream);
}
