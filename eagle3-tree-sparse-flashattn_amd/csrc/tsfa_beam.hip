// Selection over beams and vocabulary: one step of a draft (or of a beam
// search), with the beams' states put in the order of the selected parents.
//
// With x = logits[b, w, :] and c = scores[b, w],
//   value(w, v) = (c + x[v]) - lse_w,   lse_w = log sum_v exp(x[v]),
// the k best (w, v) of every b by value, ties to the lowest w * vocab + v.
// Values are formed and compared in 64 bits: with tens of candidates per unit
// of value, 32-bit rounding of lse swaps neighbours of different beams about
// once in some hundred calls.  Within a beam the order is that of the logits,
// so the vocabulary pass keeps k candidates by logit alone and needs no lse:
//   part_kernel   one workgroup per tile of a row: the tile's maximum, its sum
//                 of exponentials (64 bit) and its k best, one pass over the
//                 logits, which stay in registers;
//   merge_kernel  one workgroup per b: lse of every beam, the k best of the
//                 tiles' candidates;
//   states_kernel the states' rows of the selected parents.
// The vocabulary pass is bound by its exponentials of 64 bits (thirteen
// operations of 64 bits a logit; fp16 and fp32 logits take the same time), then
// by memory: 64 x 8 rows of 128256 fp32 logits (263 MB) take 64 us, 4.1 TB/s,
// where a copy reaches 5.1.  4 x 10 rows of fp16 (10 MB) take 12 us and 11 us of
// merge, one row of 32000 takes 6 and 8 us: there the time is that of the
// launches and of a chain of loads and barriers.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>

#include "tsfa_internal.h"

namespace tsfa {
namespace beam {

constexpr int kThreads = 256;
constexpr int kMaxK = 64;
constexpr int kMaxBeams = 256;
constexpr int kMaxStates = 8;
constexpr int64_t kStatesInside = 128 << 10;  // bytes of a sequence's selected states, see tsfa_beam_select
constexpr int64_t kMaxBlocks = 1 << 23;  // of a launch

// Statistics of one tile: maximum (as a float) and sum of exp(x - maximum).
struct PartStat {
  double sum;
  float top;
  int pad;
};

struct PartArgs {
  const void* logits;
  int64_t sb, sw;  // strides of sequence and beam, in elements
  int beams, vocab, k, tiles;
  uint64_t* keys;   // [rows][tiles][k], best first, 0: none
  PartStat* stats;  // [rows][tiles]
};

// A logit in an order of its bits that integers compare alike (-0 counts as
// 0); 0 is no candidate (-inf, NaN).
__device__ inline uint32_t order_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// A candidate of a row as one number, better = larger: its order, then the
// lower token.
__device__ inline uint64_t make_key(float x, uint32_t v) {
  const uint32_t o = order_of(x);
  return o == 0 ? 0 : ((uint64_t)o << 32) | (uint32_t)~v;
}
__device__ inline float key_logit(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ inline uint32_t key_token(uint64_t key) { return ~(uint32_t)key; }

// 2^t for -1000 < t <= 0: t = n + f, 2^f by the polynomial of degree 8 through
// the Chebyshev points of [-1/2, 1/2] (1.1e-12 off at most), n into the
// exponent.  Adding 1.5 * 2^52 rounds to n and leaves it in the low word.
__device__ inline double exp2_neg(double t) {
  constexpr double kRound = 6755399441055744.0;
  const double u = t + kRound;
  const double f = t - (u - kRound);
  double p = 1.3255224878668817e-06;
  p = fma(p, f, 1.5310079402249296e-05);
  p = fma(p, f, 0.00015403455852453838);
  p = fma(p, f, 0.0013333450568000645);
  p = fma(p, f, 0.009618129159402558);
  p = fma(p, f, 0.05550410941205933);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805459335);
  p = fma(p, f, 1.0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, u) << 52);
  return __builtin_bit_cast(double, bits);
}
constexpr double kLog2e = 1.4426950408889634074;
// exp(x - top) for x <= top, top > -inf; equal infinities weigh 1 (below -600:
// the weight at -600, which no sum notices).
__device__ inline double weight(float x, float top) {
  if (x == top) return 1.0;
  return exp2_neg(fmax((double)x - (double)top, -600.0) * kLog2e);
}

// A bound that at least k of the wave's values reach (0: no value, never
// counted), and not many more unless they tie; 1 if fewer than k are there.
// From the top bit down by counting lanes, N values to a lane.
template <int N> __device__ inline uint32_t kth_order(const uint32_t (&x)[N], int k) {
  auto count = [&](uint32_t bound) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += __builtin_popcountll(__ballot(x[i] >= bound));
    return c;
  };
  if (count(1) < k) return 1;
  uint32_t v = 0;
  for (uint32_t bit = 1u << 31; bit != 0; bit >>= 1) {
    const int c = count(v | bit);
    if (c < k) continue;
    v |= bit;
    if (c <= k + k / 2 + 4) break;
  }
  return v;
}

// EPT elements per thread, VEC of them in one 16-byte load.
template <typename T, int EPT>
__global__ __launch_bounds__(kThreads) void part_kernel(const PartArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T), NU = EPT / VEC, NW = kThreads / 64;
  extern __shared__ __attribute__((aligned(16))) uint64_t list[];  // k * EPT
  __shared__ uint32_t orders[kThreads];
  __shared__ double wsum[NW];
  __shared__ float wtop[NW];
  __shared__ uint32_t bound;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tile = blockIdx.x % a.tiles, row = blockIdx.x / a.tiles;
  const int b = row / a.beams, w = row - b * a.beams;
  const T* x = static_cast<const T*>(a.logits) + b * a.sb + w * a.sw;
  const int v0 = tile * (kThreads * EPT);

  float xs[EPT];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int v = v0 + (u * kThreads + tid) * VEC;
    if (v + VEC <= a.vocab) {
      T t[VEC];
      __builtin_memcpy(t, x + v, 16);  // rows of an odd vocabulary start anywhere
#pragma unroll
      for (int j = 0; j < VEC; ++j) xs[u * VEC + j] = (float)t[j];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) xs[u * VEC + j] = v + j < a.vocab ? (float)x[v + j] : -INFINITY;
    }
  }
  auto token = [&](int e) { return (uint32_t)(v0 + ((e / VEC) * kThreads + tid) * VEC + e % VEC); };
  if (tid == 0) count = 0;

  float mine = -INFINITY;  // fmaxf passes over NaN, which is no candidate and weighs nothing
#pragma unroll
  for (int e = 0; e < EPT; ++e) mine = fmaxf(mine, xs[e]);
  orders[tid] = order_of(mine);
  float top = mine;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
  if (lane == 0) wtop[wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) top = fmaxf(top, wtop[i]);

  // The k-th best of the threads' best elements bounds the tile's k-th best
  // from below: few more than k elements reach it, unless many tie.
  if (wave == 0) {
    uint32_t o[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) o[i] = orders[i * 64 + lane];
    const uint32_t v = kth_order(o, a.k);
    if (lane == 0) bound = v;
  }
  double sum = 0;
  if (fabsf(top) <= 4096.0f) {
    // log2 e x and log2 e top round apart: 4096 * 2^-52 at most
    const double shift = -(double)top * kLog2e;
    const float low = top - 88.0f;  // less, NaN and -inf: e^-88, which no sum notices
    double sum2 = 0;
#pragma unroll
    for (int e = 0; e < EPT; e += 2) {
      sum += exp2_neg(fma((double)fmaxf(xs[e], low), kLog2e, shift));
      sum2 += exp2_neg(fma((double)fmaxf(xs[e + 1], low), kLog2e, shift));
    }
    sum += sum2;
  } else if (top > -INFINITY) {
    // read again: kept for this loop too, they cost the kernel registers, and waves
#pragma unroll 1
    for (int e = 0; e < EPT; ++e) {
      const uint32_t v = token(e);
      const float y = v < (uint32_t)a.vocab ? (float)x[v] : -INFINITY;
      if (y > -INFINITY) sum += weight(y, top);
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
  if (lane == 0) wsum[wave] = sum;
  __syncthreads();

  const int room = a.k * EPT;
  // the bound as a logit (below every number's order: the least number)
  const float lim = bound < 0x00800000u ? -FLT_MAX : key_logit((uint64_t)bound << 32);
  if (mine >= lim) {
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      if (xs[e] >= lim) {
        const int at = atomicAdd(&count, 1);
        if (at < room) list[at] = make_key(xs[e], token(e));
      }
  }
  __syncthreads();
  int n = count;
  if (n > room) {
    // More ties at the bound than the list holds: the k-th best thread by its
    // best element's value and token, which only k threads reach, is the bound.
    auto key_of = [&](int e) {
      const uint32_t v = token(e);
      return v < (uint32_t)a.vocab ? make_key((float)x[v], v) : 0;
    };
    uint64_t best = 0;
#pragma unroll 1
    for (int e = 0; e < EPT; ++e) {
      const uint64_t key = key_of(e);
      best = key > best ? key : best;
    }
    __shared__ uint64_t bests[kThreads];
    __shared__ uint64_t exact;
    bests[tid] = best;
    if (tid == 0) {
      count = 0;
      exact = 1;
    }
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < kThreads; ++i) rank += bests[i] > best;
    if (best != 0 && rank == a.k - 1) exact = best;
    __syncthreads();
    const uint64_t by = exact;
#pragma unroll 1
    for (int e = 0; e < EPT; ++e) {
      const uint64_t key = key_of(e);
      if (key >= by) list[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    n = count;
  }
  uint64_t* out = a.keys + ((int64_t)row * a.tiles + tile) * a.k;
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t key = list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < a.k) out[rank] = key;
  }
  for (int i = n + tid; i < a.k; i += kThreads) out[i] = 0;
  if (tid == 0) {
    PartStat st;
    st.sum = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) st.sum += wsum[i];
    st.top = top;
    st.pad = 0;
    a.stats[(int64_t)row * a.tiles + tile] = st;
  }
}

// The states' rows of the parents, [batch][beams] to [batch][k].
struct States {
  const void* src[kMaxStates];
  void* dst[kMaxStates];
  int64_t row_bytes[kMaxStates];
  int n;
};
// Threads first, first + step, ... copy one row.
__device__ inline void copy_row(const States& st, int s, int64_t from, int64_t to, int64_t first, int64_t step) {
  const int64_t bytes = st.row_bytes[s];
  const char* src = static_cast<const char*>(st.src[s]) + from * bytes;
  char* dst = static_cast<char*>(st.dst[s]) + to * bytes;
  if (((reinterpret_cast<uintptr_t>(st.src[s]) | reinterpret_cast<uintptr_t>(st.dst[s]) | (uintptr_t)bytes) & 15) == 0) {
    const uint4* s16 = reinterpret_cast<const uint4*>(src);
    uint4* d16 = reinterpret_cast<uint4*>(dst);
    int64_t i = first;
    for (; i + 3 * step < bytes / 16; i += 4 * step) {
      const uint4 v0 = s16[i], v1 = s16[i + step], v2 = s16[i + 2 * step], v3 = s16[i + 3 * step];
      d16[i] = v0;
      d16[i + step] = v1;
      d16[i + 2 * step] = v2;
      d16[i + 3 * step] = v3;
    }
    for (; i < bytes / 16; i += step) d16[i] = s16[i];
  } else {
    for (int64_t i = first; i < bytes; i += step) dst[i] = src[i];
  }
}

struct MergeArgs {
  const uint64_t* keys;
  const PartStat* stats;
  const float* scores;  // [batch][beams]
  int64_t ssb, ssw;
  int beams, vocab, k, tiles;
  int64_t* tokens;
  int64_t* parents;
  float* out_scores;
  States states;  // n = 0: copied by states_kernel
};

// A candidate over all beams, better = larger value, then the lower flat = w *
// vocab + v.  The value is a double in an order of its bits that integers
// compare alike; 0 is no candidate.
struct Cand {
  uint64_t value;
  uint32_t flat, pad;
};
__device__ inline bool better(const Cand& x, const Cand& y) {
  return x.value > y.value || (x.value == y.value && x.flat < y.flat);
}
__device__ inline uint64_t value_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return u >> 63 ? ~u : u | ((uint64_t)1 << 63);
}
__device__ inline double key_value(uint64_t o) {
  return __builtin_bit_cast(double, o >> 63 ? o & ~((uint64_t)1 << 63) : ~o);
}

constexpr int kMergeThreads = 512;
constexpr int kBatch = 8;     // candidates per thread and round
constexpr int kMergeList = 1024;

__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const MergeArgs a) {
  constexpr int NW = kMergeThreads / 64;
  static_assert(kMergeList >= kMaxK * kBatch + kMaxK, "a round's candidates by rank");
  __shared__ double lse[kMaxBeams], score[kMaxBeams];
  __shared__ float tops[kMaxBeams];
  __shared__ Cand heads[kMergeThreads];
  __shared__ Cand list[2 * kMergeList];
  __shared__ Cand kept[kMaxK];
  __shared__ uint32_t wbound[NW];
  __shared__ Cand bound;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x;
  const Cand none = {0, 0xffffffffu, 0};

  // candidate c: place p of list l; the round's keys are requested ahead
  const int lists = a.beams * a.tiles;
  const int total = lists * a.k;
  const uint64_t* keys = a.keys + (int64_t)b * total;
  uint64_t raw[kBatch];
  auto request = [&](int c0) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const uint32_t c = (uint32_t)(c0 + j * kMergeThreads + tid);
      const uint32_t p = c / (uint32_t)lists, l = c - p * (uint32_t)lists;
      raw[j] = c < (uint32_t)total ? keys[(int64_t)l * a.k + p] : 0;
    }
  };
  request(0);

  // lse_w = top + log(sum) of the tiles, 16 lanes to a beam; a beam with
  // nothing above -inf, or whose score is not finite, has no candidates
  for (int w0 = 0; w0 < a.beams; w0 += kMergeThreads / 16) {
    const int w = w0 + tid / 16, l = tid & 15;
    const PartStat* st = a.stats + ((int64_t)b * a.beams + (w < a.beams ? w : a.beams - 1)) * a.tiles;
    const float c = a.scores[b * a.ssb + (w < a.beams ? w : 0) * a.ssw];
    float top = -INFINITY;
    for (int i = l; i < a.tiles; i += 16) top = fmaxf(top, st[i].top);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
    double sum = 0;
    for (int i = l; i < a.tiles; i += 16)
      if (st[i].top > -INFINITY) sum += st[i].sum * weight(st[i].top, top);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
    if (l == 0 && w < a.beams) {
      const bool alive = top > -INFINITY && c - c == 0.0f;
      tops[w] = top;
      score[w] = alive ? (double)c : -INFINITY;
      // tokens at +inf share the beam's mass: their own logit and the
      // maximum cancel
      lse[w] = top < INFINITY ? (double)top + log(sum) : log(sum);
    }
  }
  for (int i = tid; i < a.k; i += kMergeThreads) kept[i] = none;
  __syncthreads();

  // Candidates in rounds, the tiles' best first, so that the first rounds
  // bring the bound near its end and the later ones find little above it.
  for (int c0 = 0; c0 < total; c0 += kMergeThreads * kBatch) {
    const Cand last = kept[a.k - 1];
    Cand cs[kBatch], top = none;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      cs[j] = none;
      if (raw[j] != 0) {
        const uint32_t c = (uint32_t)(c0 + j * kMergeThreads + tid);
        const int w = (int)(c % (uint32_t)lists) / a.tiles;
        const float x = key_logit(raw[j]);
        const bool inf = tops[w] == INFINITY;
        if (score[w] > -INFINITY && (!inf || x == INFINITY)) {
          cs[j].value = value_key((score[w] + (inf ? 0.0 : (double)x)) - lse[w]);
          cs[j].flat = (uint32_t)w * (uint32_t)a.vocab + key_token(raw[j]);
        }
      }
      if (!better(cs[j], last)) cs[j] = none;
      if (better(cs[j], top)) top = cs[j];
    }
    if (tid == 0) count = 0;
    if (c0 + kMergeThreads * kBatch < total) request(c0 + kMergeThreads * kBatch);
    if (__syncthreads_or(top.value != 0) == 0) {
      // a round that holds one of every list: what is behind it in its list is
      // no better
      if (lists <= kMergeThreads * kBatch) break;
      continue;
    }
    // as in part_kernel, by the upper half of the value: ties stay in
    uint32_t wb;
    if (a.k <= 40) {
      const uint32_t hi[1] = {(uint32_t)(top.value >> 32)};
      wb = kth_order(hi, a.k);
    } else {
      // 64 threads' best leave too many: of all candidates (64 x 16 rows, k = 64:
      // merge 21 us, by the threads' best 35; 9 x 35 rows, k = 31: 18 and 17)
      uint32_t hi[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) hi[j] = (uint32_t)(cs[j].value >> 32);
      wb = kth_order(hi, a.k);
    }
    if (lane == 0) wbound[wave] = wb;
    __syncthreads();
    uint64_t lim = last.value > 1 ? last.value : 1;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const uint64_t v = wbound[i] > 1 ? (uint64_t)wbound[i] << 32 : 1;
      lim = v > lim ? v : lim;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (cs[j].value >= lim) {
        const int at = atomicAdd(&count, 1);
        if (at < kMergeList - kMaxK) list[at] = cs[j];
      }
    __syncthreads();
    int n = count;
    if (n > kMergeList - kMaxK) {
      // more ties than the list holds: the k-th best thread by value and
      // place, which at most k threads reach
      heads[tid] = top;
      if (tid == 0) {
        bound = last;
        count = 0;
      }
      __syncthreads();
      if (top.value != 0) {
        int rank = 0;
        for (int i = 0; i < kMergeThreads; ++i) rank += better(heads[i], top);
        if (rank == a.k - 1) bound = top;
      }
      __syncthreads();
      const Cand by = bound;
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (cs[j].value != 0 && !better(by, cs[j])) list[atomicAdd(&count, 1)] = cs[j];
      __syncthreads();
      n = count;
    }
    // the kept ones join, all are ranked, the k best stay
    for (int i = tid; i < a.k; i += kMergeThreads) list[n + i] = kept[i];
    __syncthreads();
    n += a.k;
    int base = 0;
    if (n > 2 * kMaxK) {
      // The waves' bounds leave many where k is large (ranks are a list by a
      // list: 35 beams, k = 31, 47 us of merge without this): once more by the
      // bound of all of them, which each wave finds for itself.
      uint32_t his[kMergeList / 64];
#pragma unroll
      for (int i = 0; i < kMergeList / 64; ++i)
        his[i] = i * 64 + lane < n ? (uint32_t)(list[i * 64 + lane].value >> 32) : 0;
      const uint32_t least = kth_order(his, a.k);
      if (tid == 0) count = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kMergeThreads)
        if ((uint32_t)(list[i].value >> 32) >= least) list[kMergeList + atomicAdd(&count, 1)] = list[i];
      __syncthreads();
      base = kMergeList;
      n = count;
    }
    for (int i = tid; i < n; i += kMergeThreads) {
      const Cand x = list[base + i];
      if (x.value == 0) continue;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += better(list[base + j], x);
      if (rank < a.k) kept[rank] = x;
    }
    __syncthreads();
  }
  for (int i = tid; i < a.k; i += kMergeThreads) {
    const Cand x = kept[i];
    const bool ok = x.value != 0;
    const int64_t at = (int64_t)b * a.k + i;
    const uint32_t w = ok ? x.flat / (uint32_t)a.vocab : 0;
    a.tokens[at] = ok ? (int64_t)(x.flat - w * (uint32_t)a.vocab) : 0;
    a.parents[at] = (int64_t)w;
    a.out_scores[at] = ok ? (float)key_value(x.value) : -INFINITY;
    kept[i].pad = w;
  }
  if (a.states.n == 0) return;
  __syncthreads();
  for (int s = 0; s < a.states.n; ++s)
    for (int i = wave; i < a.k; i += NW)
      copy_row(a.states, s, (int64_t)b * a.beams + kept[i].pad, (int64_t)b * a.k + i, lane, 64);
}

// States too large for the merge's one workgroup per sequence.
__global__ __launch_bounds__(kThreads) void states_kernel(const States st, const int64_t* parents, int beams, int k) {
  const int at = blockIdx.x;
  copy_row(st, blockIdx.z, (int64_t)(at / k) * beams + parents[at], at, (int64_t)blockIdx.y * kThreads + threadIdx.x,
           (int64_t)gridDim.y * kThreads);
}

// Elements of a tile per thread: long tiles, whose fixed part (reductions, the
// bound, the list) counts less and which leave the merge fewer candidates,
// where they fill the card, short ones where a row has to be spread over it.
// 128256 fp16 logits a row, the whole call: 64 x 8 rows 74 us with 64 elements,
// 79 with 32, 95 with 16; 16 x 4 rows (512 tiles of 64) 21.5 and 24; 4 x 10 rows
// (320) 23.8 and 22.1, with 8 elements 27.
inline int elements_per_thread(int64_t rows, int vocab) {
  for (int ept = 64; ept > 8; ept /= 2)
    if (rows * (((int64_t)vocab + kThreads * ept - 1) / (kThreads * ept)) >= 512) return ept;
  return 8;
}
inline int64_t tiles_of(int64_t rows, int vocab) {
  const int64_t n = (int64_t)kThreads * elements_per_thread(rows, vocab);
  return (vocab + n - 1) / n;
}

int check(int batch, int beams, int vocab, int k, int dtype) {
  if (batch < 0 || beams <= 0 || vocab <= 0 || k <= 0) return TSFA_ERR_INVALID_ARGUMENT;
  if ((int64_t)k > (int64_t)beams * vocab) return TSFA_ERR_INVALID_ARGUMENT;
  if (dtype != TSFA_DTYPE_FP16 && dtype != TSFA_DTYPE_BF16 && dtype != TSFA_DTYPE_FP32) return TSFA_ERR_UNSUPPORTED;
  if (k > kMaxK || beams > kMaxBeams || (int64_t)beams * vocab > (1 << 30)) return TSFA_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)batch * beams;
  if ((int64_t)batch * k > kMaxBlocks || rows * tiles_of(rows, vocab) > kMaxBlocks) return TSFA_ERR_UNSUPPORTED;
  return TSFA_OK;
}

template <typename T> void launch_part(const PartArgs& a, int ept, int64_t rows, hipStream_t s) {
  const dim3 grid((unsigned)(rows * a.tiles));
  const size_t lds = (size_t)a.k * ept * sizeof(uint64_t);
  if (ept == 64) hipLaunchKernelGGL((part_kernel<T, 64>), grid, dim3(kThreads), lds, s, a);
  else if (ept == 32) hipLaunchKernelGGL((part_kernel<T, 32>), grid, dim3(kThreads), lds, s, a);
  else if (ept == 16) hipLaunchKernelGGL((part_kernel<T, 16>), grid, dim3(kThreads), lds, s, a);
  else hipLaunchKernelGGL((part_kernel<T, 8>), grid, dim3(kThreads), lds, s, a);
}

}  // namespace beam
}  // namespace tsfa

using namespace tsfa;
using namespace tsfa::beam;

extern "C" size_t tsfa_beam_select_workspace_bytes(int batch, int beams, int vocab, int k) {
  if (beam::check(batch, beams, vocab, k, TSFA_DTYPE_FP32) != TSFA_OK || batch == 0) return 0;
  const int64_t rows = (int64_t)batch * beams, parts = rows * tiles_of(rows, vocab);
  return align256((size_t)parts * k * sizeof(uint64_t)) + align256((size_t)parts * sizeof(PartStat));
}

extern "C" int tsfa_beam_select(const void* logits, int64_t logits_seq_stride, int64_t logits_beam_stride,
                                const float* scores, int64_t scores_seq_stride, int64_t scores_beam_stride, int batch,
                                int beams, int vocab, int k, int dtype, int64_t* tokens, int64_t* parents,
                                float* out_scores, const void* const* states, void* const* out_states,
                                const int64_t* state_row_bytes, int n_states, void* workspace, size_t workspace_bytes,
                                tsfa_stream_t stream) {
  const int st = beam::check(batch, beams, vocab, k, dtype);
  if (st != TSFA_OK) return st;
  if (n_states < 0) return TSFA_ERR_INVALID_ARGUMENT;
  if (n_states > kMaxStates) return TSFA_ERR_UNSUPPORTED;
  if (batch == 0) return TSFA_OK;
  if (logits == nullptr || scores == nullptr || tokens == nullptr || parents == nullptr || out_scores == nullptr)
    return TSFA_ERR_INVALID_ARGUMENT;
  States sa;
  int64_t most = 0, moved = 0;
  for (int i = 0; i < n_states; ++i) {
    if (states == nullptr || out_states == nullptr || state_row_bytes == nullptr || state_row_bytes[i] < 0)
      return TSFA_ERR_INVALID_ARGUMENT;
    if (state_row_bytes[i] > 0 && (states[i] == nullptr || out_states[i] == nullptr)) return TSFA_ERR_INVALID_ARGUMENT;
    sa.src[i] = states[i];
    sa.dst[i] = out_states[i];
    sa.row_bytes[i] = state_row_bytes[i];
    most = state_row_bytes[i] > most ? state_row_bytes[i] : most;
    moved += state_row_bytes[i];
  }
  const int64_t rows = (int64_t)batch * beams;
  const int ept = elements_per_thread(rows, vocab);
  const int64_t tiles = tiles_of(rows, vocab), parts = rows * tiles;
  const size_t key_bytes = align256((size_t)parts * k * sizeof(uint64_t));
  if (workspace == nullptr || workspace_bytes < key_bytes + align256((size_t)parts * sizeof(PartStat)) ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return TSFA_ERR_WORKSPACE;

  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  PartArgs pa;
  pa.logits = logits;
  pa.sb = logits_seq_stride;
  pa.sw = logits_beam_stride;
  pa.beams = beams;
  pa.vocab = vocab;
  pa.k = k;
  pa.tiles = (int)tiles;
  pa.keys = static_cast<uint64_t*>(workspace);
  pa.stats = reinterpret_cast<PartStat*>(static_cast<char*>(workspace) + key_bytes);
  if (dtype == TSFA_DTYPE_BF16) launch_part<__bf16>(pa, ept, rows, s);
  else if (dtype == TSFA_DTYPE_FP16) launch_part<_Float16>(pa, ept, rows, s);
  else launch_part<float>(pa, ept, rows, s);

  MergeArgs ma;
  ma.keys = pa.keys;
  ma.stats = pa.stats;
  ma.scores = scores;
  ma.ssb = scores_seq_stride;
  ma.ssw = scores_beam_stride;
  ma.beams = beams;
  ma.vocab = vocab;
  ma.k = k;
  ma.tiles = (int)tiles;
  ma.tokens = tokens;
  ma.parents = parents;
  ma.out_scores = out_scores;
  // The merge's workgroup copies a sequence's states itself where they are
  // small: below 64 KB to a sequence that is as fast as a launch for them (15.7
  // to 17.0 us a call against 16.6 to 17.2) and saves the host 5 us; at 128 KB it
  // is 0.9 us slower, at 256 KB 3 us, at 1 MB 16 us.
  sa.n = n_states;
  const bool inside = moved * k <= kStatesInside;
  ma.states = sa;
  if (!inside) ma.states.n = 0;
  hipLaunchKernelGGL(merge_kernel, dim3((unsigned)batch), dim3(kMergeThreads), 0, s, ma);
  if (!inside) {
    const int64_t blocks = (most / 16 + kThreads) / kThreads;
    hipLaunchKernelGGL(states_kernel, dim3((unsigned)(batch * k), (unsigned)(blocks < 64 ? blocks : 64), (unsigned)n_states),
                       dim3(kThreads), 0, s, sa, (const int64_t*)parents, beams, k);
  }
  return hipGetLastError() == hipSuccess ? TSFA_OK : TSFA_ERR_LAUNCH;
}
