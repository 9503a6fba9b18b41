// Attention of one token per sequence over the paged cache where sequences come in groups whose first keys lie in the same
// pages (the beams of a request behind its prompt): the keys that a group shares are read once for all its rows.
//
//   out = softmax(scale * q K^T) V per head, over the keys [0, ctx) of the sequence; sinks: one more term exp(sink_h) in the
//   denominator.  A sequence without keys gets zeros.  gate: every output is multiplied by sigmoid(gate), in fp32 ahead of its one
//   rounding.
//
// A workgroup of four waves takes a cut of a range of keys for one kv head and up to 16 * RT rows: of the shared keys, rows are
// (sequence of the group, head that shares the kv head); of a sequence's own keys, the heads alone.  Every cut leaves its
// (reference, sum, accumulator) in the workspace, and `attn_beams_join_kernel` joins the cuts of a row.
//
// Blocks of 32 keys go round the waves.  For lane l, g = l / 16, r = l % 16:
//   S^T (keys x rows) = K Q^T in two tiles t of 16 keys; tile row i is key 8 (i / 4) + 4 t + i % 4, so that a lane ends up with
//     the scores of the eight neighbouring keys 8 g .. 8 g + 7 of row r;
//   O^T (d x rows) += V^T P^T: V pages hold an element's keys side by side, so a lane's eight keys of one element are one load,
//     and its probabilities are the other operand as they stand (bf16: as two numbers; fp32: v_mfma_f32_16x16x4_f32 takes them
//     key by key).
// Fragments come from the pages in this order, nothing is staged.  Lanes without a valid page read page 0 and are masked.
//
// A row's reference (what is subtracted in the exponent) is raised only when a score passes it by LAZY (in log2 units); scores,
// sums and accumulators are fp32.  bf16: a probability enters its product with V as the sum of two bf16 numbers, itself cut and
// what that leaves, 2^-15 of it off: outputs are off by the rounding of what is stored (0.0017 of their largest; rounded once,
// probabilities alone would make that up to 0.0025).  Splitting them and the second products take 0.4 of 13.5 us where the chain of a
// few blocks bounds (8 x up to 5 beams behind up to 2,900 keys), 2 of 23.5 where the vector units do most (two tiles of rows of
// heads of 64, 6 x up to 12 behind up to 5,181), and 0.3% where the bytes bound.
//
// What bounds it: the keys' bytes where there are many of them (4 x 8 beams behind 32,768 keys, 8 kv heads of 128, bf16: 552 MB in
// 105 us, 5.3 TB/s, about what a kernel that only reads reaches), otherwise the chain of loads that a workgroup begins with
// (group, lengths, page, K, V) and the second launch: 7 us for 4 beams behind 300 keys; in between, units without a share of
// the keys (12 x 16 beams of 24 heads of 128 behind 1,777: 192 workgroups walk the shared keys on 256 units, 43 us for 142 MB; fp32
// 288 on 256 units that hold one each, 94 us for 284 MB).  Against one pass per sequence, which
// reads shared keys once a beam: 16 x 8 beams behind 4,096 keys, heads of 128, 47 us and 166, heads of 64, 28 and 79.
#include <type_traits>

#include "common.h"

namespace {
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
constexpr int WAVES = 4, THREADS = WAVES * KVF_WAVE;
constexpr int BLOCK = 32;              // keys a wave takes at a time
constexpr float LAZY = 8.f;
constexpr float LOG2E = 1.4426950408889634f;

// Where two waves a SIMD are asked for, a wave has at most 256 registers.  (fp32 heads of 128 need a few more: 12 x 16 beams
// behind 1,777 keys, 24 heads, 106 us with spills, 94 with one wave a SIMD; heads of 64 in two tiles fit, 63 and 64.)
#define KVF_TWO_WAVES(FITS) __attribute__((amdgpu_waves_per_eu((FITS) ? 2 : 1)))

struct Args {
  int H, KV, G, d, bs, nb, width, q_stride, o_stride, n_seqs, n_groups;
  int blocks;          // row blocks of a group that have a workgroup of their own
  int cs, co;          // cuts of the shared keys and of a sequence's own
  float scale2;        // scale * log2(e)
  float per_group;     // 1 / (H / KV)
  unsigned bs_magic;   // floor(2^32 / bs) + 1: key / bs == mulhi(key, bs_magic) while key * bs < 2^32
};

// row / G for rows below 2^22: (row + 0.5) / G lies no nearer to a whole number than 0.5 / G, which the roundings do not reach.
__device__ __forceinline__ int group_of(int row, const Args& a) { return static_cast<int>((static_cast<float>(row) + 0.5f) * a.per_group); }

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
  // v + rest, v the probability cut to bf16.  The rest of 1 + 2^-23 of it is positive where the probability is, so that an infinite
  // value stays infinite (the sum of its products would otherwise hold inf * 0, or inf and -inf).
  struct Probs { bf16x8 v, rest; };
  static __device__ __forceinline__ Probs probs(const f32x4 (&p)[2]) {
    Probs o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t cut = __float_as_uint(p[i / 4][i % 4]) & 0xffff0000u;
      o.v[i] = __builtin_bit_cast(__bf16, static_cast<uint16_t>(cut >> 16));
      o.rest[i] = static_cast<__bf16>(fmaf(p[i / 4][i % 4], 1.f + 0x1p-23f, -__uint_as_float(cut)));
    }
    return o;
  }
  static __device__ __forceinline__ f32x4 values(const Keys& k, const Probs& p, f32x4 acc) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, p.rest, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.v, p.v, acc, 0, 0, 0);
  }
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

// The first of the sequences [first, first + n) that holds `shared` keys, from whose pages the group's are read; -1: none.
__device__ __forceinline__ int holder_of(int first, int n, int shared, const int* __restrict__ ctx_lens) {
  const int lane = threadIdx.x % KVF_WAVE;
  for (int i = 0; i < n; i += KVF_WAVE) {
    const unsigned long long held = __ballot(i + lane < n && ctx_lens[first + min(i + lane, n - 1)] >= shared);
    if (held) return first + i + __ffsll(static_cast<long long>(held)) - 1;
  }
  return -1;
}

// What a wave holds of 16 * RT rows: Q, and the running reference, sum and accumulator of each.
// FORM: WHOLE where d is 16 * DT and pages hold a multiple of 8 keys, ALIGNED where they do, ANY.
enum Form { ANY, ALIGNED, WHOLE };
template <typename T, int DT, int RT, Form FORM> struct Rows {
  typedef Frag<T> F;
  static constexpr int SLICES = DT * 16 / F::SLICE, LANE_D = F::SLICE / 4;
  // Fragments of K whose products with Q are summed in one run, whose results are then added.  (A score's error is that of
  // sums in a row: in 32 bits each fragment is four of them, and 64 in a row for heads of 256 made outputs 1.0e-6 off, 6e-7 so; heads
  // of 128 0.75e-6 and 0.45e-6.  Runs of four cost heads of 256, which have no register to spare, up to 30% of their time, runs of eight
  // 2 to 7%: 30.7 us for 8 x 8 beams behind 700 keys, 28.7 before; smaller heads nothing.)
  static constexpr int RUN = sizeof(T) == 2 || DT > 8 ? 8 : 4;
  typename F::Part q[RT][SLICES];
  f32x4 acc[RT][DT];
  float m[RT], sum[RT];
  bool live[RT];         // whether the row's sequence holds enough keys to take part

  // A lane's part of a row from element e on; behind the head's end something inside it, which `within` makes zeros (where it is
  // used: a load that is looked at is waited for).
  static __device__ __forceinline__ bool has(int j, int tiles) { return FORM == WHOLE || j < tiles; }
  static __device__ __forceinline__ typename F::Part part(const T* row, int e, int d) { return F::load(row + (FORM == WHOLE ? e : min(e, d - LANE_D))); }
  static __device__ __forceinline__ typename F::Part within(typename F::Part v, int e, int d) { return FORM == WHOLE || e < d ? v : F::zero(); }

  // Rows [row0, row0 + 16 RT) of `rows`, those of sequences of `least` keys and more: sequence first + row / G, head row % G of kv head `kvh`.
  __device__ __forceinline__ void start(const Tensors<T>& t, const Args& a, int first, int rows, int row0, int kvh, int least) {
    const int lane = threadIdx.x % KVF_WAVE, g = lane / 16, r = lane % 16, G = a.G;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = min(row0 + rt * 16 + r, rows - 1);
      const int seq = group_of(row, a);
      live[rt] = t.ctx_lens[first + seq] >= least;
      const T* from = t.q + static_cast<long>(first + seq) * a.q_stride + (kvh * G + row - seq * G) * a.d;
#pragma unroll
      for (int c = 0; c < SLICES; ++c) q[rt][c] = within(part(from, c * F::SLICE + g * LANE_D, a.d), c * F::SLICE + g * LANE_D, a.d);
      m[rt] = -INFINITY;
      sum[rt] = 0.f;
#pragma unroll
      for (int j = 0; j < DT; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Blocks kb, kb + step, ... of the keys [lo, hi) of the pages in `table`.  kb: a multiple of 8.  A block's K fragments are
  // loaded while the block before it is worked on, its page numbers looked up one earlier still: loads come back in order, so
  // one that waited for a number asked for in the same turn would wait for the V loads ahead of it too.
  __device__ __forceinline__ void walk(const Tensors<T>& t, const Args& a, const int* __restrict__ table, int kvh, int kb, int step, int lo, int hi) {
    const int lane = threadIdx.x % KVF_WAVE, g = lane / 16, r = lane % 16;
    const int d = FORM == WHOLE ? DT * 16 : a.d, tiles = d / 16;
    const long page_elems = static_cast<long>(a.KV) * a.bs * d;
    const T* kp = t.k + static_cast<long>(kvh) * a.bs * d;
    const T* vp = t.v + static_cast<long>(kvh) * a.bs * d;
    typename F::Part kf[2][SLICES];
    if (kb >= hi) return;
    // The page that holds the keys from `key` on (that of the last key behind it).  No load depends on whether there are
    // more keys, the last turn is one of its own: behind a branch around loads the compiler waits as if they were not asked for.
    const int last = FORM != ANY ? page_of(hi - 1, a) : 0;
    auto lookup = [&](int key) { return table[min(page_of(key, a), last)]; };
    auto valid = [&](int page) { return page >= 0 && page < a.nb; };
    auto load_k = [&](int at, int page) {         // page (not for ANY): that of the keys at + 8 (r / 4)
      if constexpr (FORM != ANY) {
        const int key = at + 8 * (r / 4);
        const bool ok = key < hi && valid(page);
        const T* from = kp + (ok ? page : 0) * page_elems + static_cast<long>((ok ? key - page_of(key, a) * a.bs : 0) + r % 4) * d;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int c = 0; c < SLICES; ++c) kf[tt][c] = part(from + tt * 4 * d, c * F::SLICE + g * LANE_D, d);
      } else {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int key = at + 8 * (r / 4) + 4 * tt + r % 4;
          const int p = key < hi ? table[key / a.bs] : -1;
          const T* from = kp + (valid(p) ? p : 0) * page_elems + static_cast<long>(valid(p) ? key % a.bs : 0) * d;
#pragma unroll
          for (int c = 0; c < SLICES; ++c) kf[tt][c] = part(from, c * F::SLICE + g * LANE_D, d);
        }
      }
    };
    int pv = 0, pk_next = 0, pv_next = 0;       // (not for ANY) the pages of keys kb + 8 g, next + 8 (r / 4), next + 8 g
    if constexpr (FORM != ANY) {
      const int pk = lookup(kb + 8 * (r / 4));
      pv = lookup(kb + 8 * g);
      pk_next = lookup(kb + step + 8 * (r / 4));
      pv_next = lookup(kb + step + 8 * g);
      asm volatile("" : "+v"(pk_next), "+v"(pv_next));       // (to have them ahead of K, not where the loop begins)
      load_k(kb, pk);
    } else {
      load_k(kb, 0);
    }
    auto turn = [&](auto more) {        // more: there is a further block
      const int next = kb + step;
      typename F::Keys vf[DT];
      unsigned keep = 0;                // which of the lane's keys kb + 8 g + (0 .. 7) count
      int pk_after = 0, pv_after = 0;
      if constexpr (FORM != ANY) {
        const int key = kb + 8 * g, from = max(lo - key, 0), to = min(hi - key, 8);
        const bool ok = key < hi && valid(pv);
        keep = ok && to > from ? (0xffu >> (8 - to)) & (0xffu << from) : 0u;
        const T* v0 = vp + (ok ? pv : 0) * page_elems + (ok ? key - page_of(key, a) * a.bs : 0) + r * a.bs;
        if constexpr (more) {
          pk_after = lookup(next + step + 8 * (r / 4));
          pv_after = lookup(next + step + 8 * g);
        }
#pragma unroll
        for (int j = 0; j < DT; ++j)
          vf[j] = F::load_keys(v0 + static_cast<long>(has(j, tiles) ? j : 0) * 16 * a.bs);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = kb + 8 * g + i;
          const int p = key >= lo && key < hi ? table[key / a.bs] : -1;
          keep |= valid(p) ? 1u << i : 0u;
          const T* v0 = vp + (valid(p) ? p : 0) * page_elems + (valid(p) ? key % a.bs : 0) + r * a.bs;
#pragma unroll
          for (int j = 0; j < DT; ++j)
            F::set(vf[j], i, v0[static_cast<long>(has(j, tiles) ? j : 0) * 16 * a.bs]);
        }
      }
      const bool whole = __all(keep == 0xffu);
      f32x4 s[RT][2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int c0 = 0; c0 < SLICES; c0 += RUN) {
            f32x4 run = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = c0; c < min(c0 + RUN, SLICES); ++c) run = F::scores(within(kf[tt][c], c * F::SLICE + g * LANE_D, d), q[rt][c], run);
            s[rt][tt] = c0 ? s[rt][tt] + run : run;
          }
        }
      if constexpr (more) load_k(next, pk_next);
      // All products are read here, ahead of any branch: in a form of this loop where the first read of a product of the matrix cores
      // stood behind the meeting of two branches, one of them long, hipcc 7.2 put no wait ahead of it, and scores were wrong.
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float x = s[rt][i / 4][i % 4] * a.scale2;
          asm volatile("" : "+v"(x));
          s[rt][i / 4][i % 4] = x;
        }
      typename F::Probs pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!whole)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[rt][i / 4][i % 4] = keep >> i & 1u ? s[rt][i / 4][i % 4] : -INFINITY;
        float most = s[rt][0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, s[rt][i / 4][i % 4]);
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
          p[i / 4][i % 4] = __builtin_amdgcn_exp2f(s[rt][i / 4][i % 4] - ref);
          sum[rt] += p[i / 4][i % 4];
        }
        pf[rt] = F::probs(p);
      }
      if (!whole)
#pragma unroll
        for (int j = 0; j < DT; ++j) F::clear(vf[j], keep);
#pragma unroll
      for (int j = 0; j < DT; ++j)        // (those behind the head's end too: nobody reads their sums)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][j] = F::values(vf[j], pf[rt], acc[rt][j]);
      kb = next;
      pv = pv_next;
      pk_next = pk_after;
      pv_next = pv_after;
    };
    while (kb + step < hi) turn(std::true_type{});
    turn(std::false_type{});
  }

  // Where row rt * 16 + r of the rows leaves its results as cut `cut`; -1: nowhere.
  __device__ __forceinline__ long place(const Args& a, int rt, int first, int rows, int row0, int kvh, int cut) const {
    const int r = threadIdx.x % 16, G = a.G, row = row0 + rt * 16 + r, seq = group_of(row, a);
    return row < rows ? (static_cast<long>(first + seq) * a.H + kvh * G + row - seq * G) * (a.cs + a.co) + cut : -1;
  }
  // (reference, sum over all keys of the cut), -inf where there are none (NaN stays NaN); whether there is an accumulator.
  __device__ __forceinline__ bool leave_sum(const Tensors<T>& t, int rt, long at, float top, float total, bool writes) const {
    const bool any = live[rt] && (total > 0.f || total != total);
    if (writes && at >= 0) t.ml[at] = any ? make_float2(top > -INFINITY ? top : 0.f, total) : make_float2(-INFINITY, 0.f);
    return any && at >= 0;
  }
  __device__ __forceinline__ float whole_sum(int rt) const {
    float l = sum[rt];
    l += __shfl_xor(l, 16, KVF_WAVE);
    return l + __shfl_xor(l, 32, KVF_WAVE);
  }
};

// Cut `c` of `n` of the keys [lo, hi), in whole rounds of `round` keys.
__device__ __forceinline__ void cut_of(int& lo, int& hi, int c, int n, int round) {
  const int first = lo & ~7;
  const int per = ((hi - first + n - 1) / n + round - 1) / round * round;
  const int from = first + min(c * per, hi - first), to = min(from + per, hi);
  lo = max(lo, from);
  hi = to;
}

// The workgroups of the first n_groups * cs * blocks * KV numbers take a cut of a group's shared keys, the four waves a block
// each in turn; of the others every wave takes a cut of a sequence's own keys by itself.  The kv head is the fastest index:
// workgroups go to the eight XCDs in turn, so with eight heads an L2 holds the keys of one, also for a group's further rows.
template <typename T, int DT, int RT, Form FORM>
__global__ __launch_bounds__(THREADS) KVF_TWO_WAVES(sizeof(T) == 2 ? RT * DT <= 16 && DT < 16 : RT * DT <= 8 && DT < 8) void attn_beams_kernel(Tensors<T> t, Args a) {
  __shared__ f32x4 lds_acc[RT][DT][WAVES - 1][KVF_WAVE];
  __shared__ float2 lds_ml[RT][WAVES][16];
  const int shared_items = a.n_groups * a.cs * a.blocks * a.KV;
  const int G = a.G, most = a.width * a.bs, lane = threadIdx.x % KVF_WAVE, wave = threadIdx.x / KVF_WAVE, g = lane / 16, r = lane % 16;
  if (static_cast<int>(blockIdx.x) < shared_items) {
    const int item = blockIdx.x;
    const int kvh = item % a.KV, block = item / a.KV % a.blocks, cut = item / a.KV / a.blocks % a.cs, group = item / a.KV / a.blocks / a.cs;
    const int first = min(max(t.cu_groups[group], 0), a.n_seqs), n = min(max(t.cu_groups[group + 1], first), a.n_seqs) - first;
    if (n == 0) return;
    const int rows = n * G, tiles = a.d / 16;
    int lo = 0, hi = min(max(t.shared_lens[group], 0), most);
    const int shared = max(hi, 1), holder = holder_of(first, n, shared, t.ctx_lens);
    if (holder < 0) hi = 0;
    cut_of(lo, hi, cut, a.cs, WAVES * BLOCK);
    for (int row0 = block * 16 * RT; row0 < rows; row0 += a.blocks * 16 * RT) {
      typedef Rows<T, DT, RT, FORM> Held;
      Held x;
      x.start(t, a, first, rows, row0, kvh, shared);
      x.walk(t, a, t.table + static_cast<long>(max(holder, 0)) * a.width, kvh, lo + wave * BLOCK, WAVES * BLOCK, lo, hi);
      // the waves' results: tile j of the elements is summed by wave j % WAVES
      float l[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        l[rt] = x.whole_sum(rt);
        if (lane < 16) lds_ml[rt][wave][r] = make_float2(x.m[rt], l[rt]);
      }
      __syncthreads();
      long at[RT];
      bool any[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_ml[rt][w][r].x);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          const float2 o = lds_ml[rt][w][r];
          total += o.x > -INFINITY || o.y != o.y ? o.y * __builtin_amdgcn_exp2f(o.x - top) : 0.f;
        }
        const float by = x.m[rt] > -INFINITY ? __builtin_amdgcn_exp2f(x.m[rt] - top) : 0.f;
        at[rt] = x.place(a, rt, first, rows, row0, kvh, cut);
        any[rt] = x.leave_sum(t, rt, at[rt], top, total, wave == 0 && lane < 16);
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          x.acc[rt][j] *= by;
          if (j % WAVES != wave && Held::has(j, tiles)) lds_acc[rt][j][wave < j % WAVES ? wave : wave - 1][lane] = x.acc[rt][j];
        }
      }
      __syncthreads();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int j = 0; j < DT; ++j)
          if (j % WAVES == wave && Held::has(j, tiles)) {
            f32x4 o = x.acc[rt][j];
#pragma unroll
            for (int w = 0; w < WAVES - 1; ++w) o += lds_acc[rt][j][w][lane];
            if (any[rt]) *reinterpret_cast<f32x4*>(t.acc + at[rt] * a.d + j * 16 + g * 4) = o;
          }
    }
  } else {
    // (no barrier from here on)
    const int item = (blockIdx.x - shared_items) * WAVES + wave;
    const int kvh = item % a.KV, cut = item / a.KV % a.co, seq = item / a.KV / a.co;
    if (seq >= a.n_seqs) return;
    typedef Rows<T, DT, 1, FORM> Held;
    Held x;
    x.start(t, a, seq, G, 0, kvh, 1);        // (loaded while the group is looked for)
    const int ctx = t.ctx_lens[seq];
    // the group that the sequence is in
    int lo = 0;
    bool grouped = false;
    for (int g0 = 0; g0 < a.n_groups && !grouped; g0 += KVF_WAVE) {
      const int g = min(g0 + lane, a.n_groups - 1);
      const unsigned long long here = __ballot(t.cu_groups[g] <= seq && seq < t.cu_groups[g + 1]);
      if (here) {
        if (a.cs) lo = min(max(t.shared_lens[min(g0 + __ffsll(static_cast<long long>(here)) - 1, a.n_groups - 1)], 0), most);
        grouped = true;
      }
    }
    if (!grouped && cut == 0)       // nobody else tells of its shared keys
      for (int i = lane; i < G * a.cs; i += KVF_WAVE)
        t.ml[(static_cast<long>(seq) * a.H + kvh * G + i / a.cs) * (a.cs + a.co) + i % a.cs] = make_float2(-INFINITY, 0.f);
    int hi = max(min(ctx, most), 0);
    if (lo > hi) lo = 0;          // shorter than what its group shares: all of its keys are its own
    cut_of(lo, hi, cut, a.co, BLOCK);
    for (int row0 = 0; row0 < G; row0 += 16) {
      if (row0) x.start(t, a, seq, G, row0, kvh, 1);
      x.walk(t, a, t.table + static_cast<long>(seq) * a.width, kvh, lo & ~7, BLOCK, lo, hi);
      const long at = x.place(a, 0, seq, G, row0, kvh, a.cs + cut);
      const float total = x.whole_sum(0);       // (all lanes take part)
      if (x.leave_sum(t, 0, at, x.m[0], total, g == 0))
#pragma unroll
        for (int j = 0; j < DT; ++j)
          if (Held::has(j, a.d / 16)) *reinterpret_cast<f32x4*>(t.acc + at * a.d + j * 16 + g * 4) = x.acc[0][j];
    }
  }
}

__device__ __forceinline__ float wave_of(float v, bool sum) {
  auto with = [&](float other) { v = sum ? v + other : fmaxf(v, other); };
  with(dpp_move<0xB1>(v));        // lane ^ 1
  with(dpp_move<0x4E>(v));        // lane ^ 2
  with(dpp_move<0x141>(v));       // the other four of 8 lanes
  with(dpp_move<0x140>(v));       // the other eight of 16
  with(__shfl_xor(v, 16, KVF_WAVE));
  with(__shfl_xor(v, 32, KVF_WAVE));
  return v;
}

// The cuts' sums and accumulators of a row at the largest of their references.  A wave takes a row, or with PARTS waves each
// every so many of its cuts (the whole pass, bf16, heads of 64, a wave and four: 2 x 8 beams behind 9,000 keys in 38 cuts 10.4 and
// 9.6 us, 3 x 4 behind 1,500 in 8 cuts, fp32, 10.3 and 11.1).  Lanes: four elements each, of up to four cuts side by side.
template <typename T, int PARTS, bool GATED>
__global__ __launch_bounds__(THREADS) void attn_beams_join_kernel(const float* acc, const float2* ml, T* __restrict__ out,
                                                                  const float* sinks, const T* __restrict__ gate, int gate_stride, Args a) {
  __shared__ f32x4 lds[WAVES][KVF_WAVE];
  const int lane = threadIdx.x % KVF_WAVE, wave = threadIdx.x / KVF_WAVE, cuts = a.cs + a.co;
  const int part = wave % PARTS;
  const long last = static_cast<long>(a.n_seqs) * a.H - 1, want = static_cast<long>(blockIdx.x) * (WAVES / PARTS) + wave / PARTS;
  if (PARTS == 1 && want > last) return;
  const long row = want;       // (PARTS > 1: as many workgroups as rows)
  const int h = static_cast<int>(row % a.H);
  const float2* mine = ml + row * cuts;
  const int quads = a.d / 4, side = quads > 32 ? 1 : quads > 16 ? 2 : 4;
  const int sub = lane / (KVF_WAVE / side), at = lane % (KVF_WAVE / side);
  // accumulators of U cuts in flight, the first ahead of everything else; one without keys has left none: what is read in its
  // place is not used
  constexpr int U = 4;
  const int step = side * PARTS;
  const float* from = acc + row * cuts * a.d + min(at, quads - 1) * 4;
  f32x4 v[U];
  float2 x[U];
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + u * step, cuts - 1);
      x[u] = mine[c];
      v[u] = *reinterpret_cast<const f32x4*>(from + static_cast<long>(c) * a.d);
    }
  };
  const int first = sub * PARTS + part;
  load(first);
  f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (GATED)
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = Elem<T>::load(gate + row / a.H * gate_stride + static_cast<long>(h) * a.d + min(at, quads - 1) * 4 + i);
  const float2 none = make_float2(-INFINITY, 0.f);
  const float2 one = lane < cuts ? mine[lane] : none, two = lane + KVF_WAVE < cuts ? mine[lane + KVF_WAVE] : none;
  const float sink = sinks != nullptr ? sinks[h] * LOG2E : -INFINITY;
  float top = wave_of(fmaxf(one.x, two.x), false);
  const bool any = top > -INFINITY;
  top = fmaxf(top, sink);
  const float ref = top > -INFINITY ? top : 0.f;
  auto weight = [&](float m) { return __builtin_amdgcn_exp2f(m - ref); };      // 0 of -inf
  float total = (one.x > -INFINITY ? one.y * weight(one.x) : 0.f) + (two.x > -INFINITY ? two.y * weight(two.x) : 0.f);
  total = wave_of(total, true) + weight(sink);
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c0 = first; c0 < cuts; c0 += U * step) {
    if (c0 != first) load(c0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * step < cuts && x[u].x > -INFINITY) o += v[u] * weight(x[u].x);
  }
  for (int s = KVF_WAVE / side; s < KVF_WAVE; s *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], s, KVF_WAVE);
  if constexpr (PARTS > 1) {
    static_assert(PARTS == WAVES, "a row a workgroup");
    lds[wave][lane] = o;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) o += lds[w][lane];
  }
  if (sub == 0 && at < quads) {
    T* to = out + row / a.H * a.o_stride + static_cast<long>(h) * a.d + at * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = any ? o[i] / total : 0.f;
      Elem<T>::store(to + i, GATED ? x / (1.f + expf(-z[i])) : x);
    }
  }
}

// Heads up to so many elements have room for two tiles of rows a wave, and for two waves a SIMD.
template <typename T> constexpr int TWO_TILES = sizeof(T) == 2 ? 128 : 64;
int row_tiles_of(int bf16, int d, int bs, int rows) { return rows > 16 && d <= (bf16 ? TWO_TILES<bf16_t> : TWO_TILES<float>) && bs % 8 == 0 ? 2 : 1; }

template <typename T, int DT, int RT, Form FORM>
int launch(const Tensors<T>& t, const Args& a, hipStream_t stream) {
  const long items = static_cast<long>(a.n_groups) * a.cs * a.blocks * a.KV + (static_cast<long>(a.n_seqs) * a.co * a.KV + WAVES - 1) / WAVES;
  if (items * WAVES > 0x7fffffffL) return static_cast<int>(hipErrorInvalidValue);
  attn_beams_kernel<T, DT, RT, FORM><<<dim3(static_cast<unsigned>(items)), THREADS, 0, stream>>>(t, a);
  return kvf_last_error();
}
template <typename T, int DT> int launch_form(const Tensors<T>& t, const Args& a, int row_tiles, hipStream_t stream) {
  if (a.bs % 8) return launch<T, DT, 1, ANY>(t, a, stream);
  if constexpr (DT <= TWO_TILES<T> / 16)
    if (row_tiles == 2) return a.d == DT * 16 ? launch<T, DT, 2, WHOLE>(t, a, stream) : launch<T, DT, 2, ALIGNED>(t, a, stream);
  return a.d == DT * 16 ? launch<T, DT, 1, WHOLE>(t, a, stream) : launch<T, DT, 1, ALIGNED>(t, a, stream);
}
template <typename T> int launch_dims(const Tensors<T>& t, const Args& a, int row_tiles, hipStream_t stream) {
  if (a.d <= 32) return launch_form<T, 2>(t, a, row_tiles, stream);
  if (a.d <= 64) return launch_form<T, 4>(t, a, row_tiles, stream);
  if (a.d <= 96) return launch_form<T, 6>(t, a, row_tiles, stream);
  if (a.d <= 128) return launch_form<T, 8>(t, a, row_tiles, stream);
  return launch_form<T, 16>(t, a, row_tiles, stream);
}
constexpr int JOIN_WIDE = 16;     // more cuts of a row than so many are joined by four waves

template <typename T>
int run(const void* q, const void* k, const void* v, const int* table, const int* cu_groups, const int* shared_lens, const int* ctx_lens,
        void* out, float* acc, void* ml, const float* sinks, const void* gate, int gate_stride, const Args& a, int row_tiles, hipStream_t stream) {
  const Tensors<T> t{static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), table, cu_groups, shared_lens, ctx_lens,
                     acc, static_cast<float2*>(ml)};
  const int rc = launch_dims<T>(t, a, row_tiles, stream);
  if (rc) return rc;
  const long rows = static_cast<long>(a.n_seqs) * a.H;
  auto join = [&](auto parts, auto gated, long groups) {
    attn_beams_join_kernel<T, decltype(parts)::value, decltype(gated)::value><<<static_cast<unsigned>(groups), THREADS, 0, stream>>>(
        acc, static_cast<const float2*>(ml), static_cast<T*>(out), sinks, static_cast<const T*>(gate), gate_stride, a);
  };
  auto join_rows = [&](auto gated) {
    if (a.cs + a.co > JOIN_WIDE && rows <= 0x7fffffffL / THREADS) join(std::integral_constant<int, WAVES>{}, gated, rows);
    else join(std::integral_constant<int, 1>{}, gated, (rows + WAVES - 1) / WAVES);
  };
  if (gate != nullptr) join_rows(std::true_type{});
  else join_rows(std::false_type{});
  return kvf_last_error();
}
}  // namespace

// Tiles of 16 rows that a workgroup takes where a group has `rows` rows a kv head.
KVF_EXPORT int kvf_attn_beams_row_tiles(int bf16, int d, int bs, int rows) { return row_tiles_of(bf16, d, bs, rows); }

// q [n_seqs] rows of H heads; pages k [nb, KV, bs, d], v [nb, KV, d, bs]; table [n_seqs, width]; cu_groups [n_groups + 1];
// shared_lens [n_groups]; ctx_lens [n_seqs]; gate: null, or [n_seqs] rows of H * d elements, gate_stride apart.  Workspace: acc [n_seqs, H, cs + co, d], ml [n_seqs, H, cs + co, 2].
KVF_EXPORT int kvf_attn_beams(int bf16, const void* q, const void* k, const void* v, const int* table, const int* cu_groups,
                              const int* shared_lens, const int* ctx_lens, void* out, float* acc, void* ml, const float* sinks,
                              const void* gate, int gate_stride, int H,
                              int KV, int d, int bs, int nb, int width, int q_stride, int o_stride, int n_seqs, int n_groups, int widest,
                              int cs, int co, float scale, hipStream_t stream) {
  if (KV < 1 || H < KV || H % KV || d < 16 || d > 256 || d % 16 || bs < 1 || nb < 1 || width < 0 || n_seqs < 0 || n_groups < 0 ||
      widest < 1 || cs < 0 || co < 1 || cs > 64 || co > 64 || (n_groups == 0 && cs))
    return static_cast<int>(hipErrorInvalidValue);
  if (static_cast<long>(width) * bs >= 1L << 30 || static_cast<long>(width) * bs * bs >= (1L << 32)) return static_cast<int>(hipErrorInvalidValue);
  if (gate != nullptr && gate_stride < H * d && n_seqs > 1) return static_cast<int>(hipErrorInvalidValue);
  if (n_seqs == 0) return 0;
  const long rows = static_cast<long>(widest) * (H / KV);
  if (rows > 1 << 20 || static_cast<long>(n_seqs) * (H / KV) >= 1 << 22) return static_cast<int>(hipErrorInvalidValue);
  const int row_tiles = row_tiles_of(bf16, d, bs, static_cast<int>(rows)), blocks = static_cast<int>((rows + 16 * row_tiles - 1) / (16 * row_tiles));
  const Args a{H, KV, H / KV, d, bs, nb, width, q_stride, o_stride, n_seqs, n_groups, blocks, cs, co, scale * LOG2E, 1.f / static_cast<float>(H / KV),
               bs > 1 ? static_cast<unsigned>((1ull << 32) / bs) + 1u : 0u};
  return bf16 ? run<bf16_t>(q, k, v, table, cu_groups, shared_lens, ctx_lens, out, acc, ml, sinks, gate, gate_stride, a, row_tiles, stream)
              : run<float>(q, k, v, table, cu_groups, shared_lens, ctx_lens, out, acc, ml, sinks, gate, gate_stride, a, row_tiles, stream);
}
