// Tree attention over a paged K/V pool for sequences of different lengths:
// packed queries, every sequence with its own query and key count, read on
// the device.
//
// For token i of a sequence with q query tokens and n keys (its query tokens'
// own keys the last q of them, P = n - q before),
//   O = softmax(scale * Q K^T) V over the keys it sees: the P prefix keys, and
//   key P + j iff tree_mask[i][j] (j <= i without a mask).
// A row that sees no key is 0 (its LSE -inf): such rows pad a batch, and a NaN
// there would enter the pool with the next layer's keys.
//
// One workgroup per CU takes an equal run of the call's steps (tsfa_paged.h);
// what the run's first and last tile share with the neighbours' goes through
// the workspace, in fp32, and combine_kernel joins it.  A workgroup's waves
// are S key streams of RG row groups of 32 rows; a step is 32 S keys, of which
// stream s takes 32 through its own LDS ring (global_load_lds, HBM -> LDS
// without registers).  Three shapes, chosen in sizes_of:
//   S = 4, RG = 1   32 rows: decoding and little work, every wave on keys of
//                   its own, the streams joined in LDS;
//   S = 2, RG = 4   128 rows: trees, four waves share each key;
//   S = 1, RG = 8   256 rows: much work, K and V read half as often; half of a
//                   SIMD's waves run one product behind the others.
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: a lane holds one query
// row in both, so the softmax statistics stay in the lane, with one exchange
// between the lane halves.
//
// What bounds it: with 32 rows the reading of K and V (64 sequences of 500 to
// 16384 keys, one token each: 1.17 GB in 223 us, 5.2 TB/s, a copy's rate); with
// 128 rows the reading of K and V for each of them and the issue of matrix
// products beside the softmax, with 256 the issue alone (4 x 200 to 256 tokens of
// 64 heads by 8192 to 32768 keys: 472 GFLOP in 520 us, 900 TFLOP/s, where a large
// product reaches 1170 to 1220; MFMA busy 50 % at a power-limited clock); in
// calls of a few steps the fixed part, 8 us until a run's first unit has arrived
// and 3 to 8 us for the partial tiles' store and join.
#include <hip/hip_runtime.h>

#include <math.h>

#include <atomic>
#include <type_traits>

#include "tsfa_internal.h"
#include "tsfa_paged.h"

namespace tsfa {
namespace varlen {

using paged::Cut;
using paged::Place;
using paged::Seq;

using paged::kTableIds;
using paged::kTreeUnits;
constexpr float kRescaleLog2 = 8.0f;

struct Args {
  const void* q;
  const void* cache;
  void* out;
  float* lse;              // [total_q][num_heads] or null
  const uint8_t* mask;     // nonzero: visible; null: causal
  int64_t mask_seq, mask_row;
  int mask_n;              // rows and columns of the mask
  paged::Seqs seqs;
  Cut cut;
  int64_t sqn, sqh, son, soh;      // elements
  int64_t cp, cs, cr, ch;          // cache: page, K/V slot, row, head
  float scale_log2;                // |sm_scale| * log2(e), never 0
  int neg_q;                       // sm_scale < 0: Q enters negated
  int num_heads, groups;           // workgroups on the line
  float4* ws_o;                    // [2 * groups][RG][D / 8][64] unnormalised O, a lane's registers in order
  float2* ws_ml;                   // [2 * groups][rows] (m, l)
  int* ws_runs;                    // [groups] runs on which the tile that starts in the run ends (0: within it)
  // [groups] that tile: its sequence's query rows, kv head, tile, place on the
  // line, a run's length
  struct Desc {
    int q0, q_len, kvh, tile;
    int64_t at, per;
  };
  Desc* ws_desc;
};

// Layout of 32-key tiles of D elements: key row k, 16-byte chunk c at chunk
// c ^ swz(k), so that the operand reads below spread over the LDS banks.
template <int D> __device__ inline int swz_k(int key) { return D == 128 ? (key & 15) : ((key >> 1) & 7); }
template <int D> __device__ inline int swz_v(int key) { return D == 128 ? ((key & 3) << 2) : (((key >> 1) & 1) << 2); }

template <typename V, typename U> __device__ inline V bit_cast(U u) { return __builtin_bit_cast(V, u); }
__device__ inline uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const TSFA_LDS void*)p; }

// 64 lanes x 16 bytes HBM -> LDS lds .. lds + 1023, lane i from base + off.
// In inline asm so that the compiler does not make every LDS read wait for
// it; vm_wait orders it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved; the clobber documents the write
__device__ inline void dma_1k(const void* base, uint32_t off, uint32_t lds_in) {
  const uint64_t u = reinterpret_cast<uint64_t>(base);
  const uint64_t sbase = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32)) << 32) |
                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_in);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(sbase), "s"(lds)
               : "memory", "m0");
}
// The same with an address per lane.
__device__ inline void dma_1k_rows(const void* src, uint32_t lds_in) {
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_in);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}
// N such loads to consecutive LDS KBs from one base: load i reads base +
// off[i] + i KB (the immediate offset counts for both addresses).
template <int N> __device__ inline void dma_rows(const void* base, const uint32_t (&off)[N], uint32_t lds_in) {
  static_assert(N == 1 || N == 2 || N == 4, "up to 16 key rows");
  const uint64_t u = reinterpret_cast<uint64_t>(base);
  const uint64_t sbase = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32)) << 32) |
                         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_in);
  if constexpr (N == 4)
    asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %0, %4\n\tglobal_load_lds_dwordx4 %1, %4 offset:0x400\n\t"
                 "global_load_lds_dwordx4 %2, %4 offset:0x800\n\tglobal_load_lds_dwordx4 %3, %4 offset:0xc00"
                 :
                 : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(sbase), "s"(lds)
                 : "memory", "m0");
  else if constexpr (N == 1)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(off[0]), "s"(sbase), "s"(lds)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %0, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400"
                 :
                 : "v"(off[0]), "v"(off[1]), "s"(sbase), "s"(lds)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
// max(a, b, c) in one instruction (fmaxf first quiets operands the compiler
// cannot prove canonical, one more instruction each).
__device__ inline float max3f(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The largest of 16 scores.  One block: between blocks the compiler waits a
// cycle for what it cannot see in them.  It cannot see either that a matrix
// product may just have written them: FRESH waits for that (11 cycles).
template <bool FRESH> __device__ inline float max16f(const f32x16& s) {
  float r, t0, t1, t2, t3;
  if constexpr (FRESH) asm volatile("s_nop 15" ::"v"(s));
  asm volatile(
      "v_max3_f32 %0, %5, %6, %7\n\tv_max3_f32 %1, %8, %9, %10\n\tv_max3_f32 %2, %11, %12, %13\n\t"
      "v_max3_f32 %3, %14, %15, %16\n\tv_max3_f32 %4, %17, %18, %19\n\tv_max3_f32 %0, %0, %1, %20\n\t"
      "v_max3_f32 %2, %2, %3, %4\n\tv_max_f32 %0, %0, %2"
      : "=&v"(r), "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(s[0]), "v"(s[1]), "v"(s[2]), "v"(s[3]), "v"(s[4]), "v"(s[5]), "v"(s[6]), "v"(s[7]), "v"(s[8]), "v"(s[9]),
        "v"(s[10]), "v"(s[11]), "v"(s[12]), "v"(s[13]), "v"(s[14]), "v"(s[15]));
  return r;
}
template <int N> __device__ inline void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
// At most `left` units of LPW loads each still on their way (left <= K).
template <int LPW, int K> __device__ inline void wait_units(int left) {
  if constexpr (K == 0) {
    vm_wait<0>();
  } else {
    if (left >= K) vm_wait<K * LPW>();
    else wait_units<LPW, K - 1>(left);
  }
}
__device__ inline void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// The same among the waves of a stream; ALONE: one wave, which waits for what
// it reads.
template <bool ALONE> __device__ inline void stream_barrier() {
  if constexpr (ALONE) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  else barrier();
}

__device__ inline int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ inline int64_t readlane64(int64_t x, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, l);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)x >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// x of the lane that the DPP control names, 0 where there is none.
template <int CTRL, int ROWS> __device__ inline int64_t dpp64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)((uint64_t)x >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// Sums over the lanes up to each one, without LDS: shifts within rows of 16,
// then the last lane of row 0 (2) to row 1 (3), of row 1 to rows 2 and 3.
__device__ inline int64_t lane_scan(int64_t x) {
  x += dpp64<0x111, 0xf>(x);
  x += dpp64<0x112, 0xf>(x);
  x += dpp64<0x114, 0xf>(x);
  x += dpp64<0x118, 0xf>(x);
  x += dpp64<0x142, 0xa>(x);
  x += dpp64<0x143, 0xc>(x);
  return x;
}

// The sequences in a wave's registers, lane l holding sequence b0 + l.
struct LaneSeqs {
  int b0;
  int q0, q_len, kv_len, list;
  // loads and returns the line up to and including each lane's sequence
  __device__ int64_t load(const paged::Seqs& s, const Cut& c, int from, int lane) {
    b0 = from;
    Seq mine{};
    if (b0 + lane < s.batch) mine = paged::seq_of(s, b0 + lane);
    q0 = mine.q0;
    q_len = mine.q_len;
    kv_len = mine.kv_len;
    list = mine.list;
    return lane_scan(paged::head_length(c, mine) * c.num_kv_heads);
  }
  __device__ Seq at(int l) const {
    Seq r;
    r.q0 = __builtin_amdgcn_readlane(q0, l);
    r.q_len = __builtin_amdgcn_readlane(q_len, l);
    r.kv_len = __builtin_amdgcn_readlane(kv_len, l);
    r.prefix = max(r.kv_len - r.q_len, 0);
    r.list = __builtin_amdgcn_readlane(list, l);
    r.pages = 0;  // kv_len lies within them
    return r;
  }
};

// The logical run of a workgroup: neighbouring runs share K/V units, so the
// runs are dealt to the 8 XCDs (block id modulo 8) in contiguous eighths.
__device__ inline int run_of_block(int block, int groups) {
  return groups % 8 == 0 ? (block % 8) * (groups / 8) + block / 8 : block;
}

template <int D, int S, int RG> struct Shape {
  static constexpr int kWaves = S * RG;
  static constexpr int kRows = 32 * RG;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTile = 32 * kRowBytes;             // K or V of a unit
  static constexpr int kUnit = 2 * kTile;                  // ring stage: K, then V
  static constexpr int kStages = 131072 / (S * kUnit);     // 128 KB of rings
  static constexpr int kLpw = kUnit / 1024 / RG;           // 1 KB loads of a wave per unit
  static constexpr int kRing = S * kStages * kUnit;
  static constexpr int kWords = kTreeUnits * kRows * 4;
  // Q's way in: its rows fill the last kQStages stages of every ring before
  // these are first used, so kAhead units are requested beside it
  static constexpr int kQBytes = kRows * kRowBytes;
  static constexpr int kQStages = (kQBytes + S * kUnit - 1) / (S * kUnit);
  static constexpr int kQLoads = kQBytes / 1024 / kWaves;
  static constexpr int kAhead = kStages - (kQStages > (S == 1 ? 2 : 1) ? kQStages : (S == 1 ? 2 : 1));
  static constexpr int kLds = kRing + kTableIds * 8 + kWords;
};

// LDS byte of Q's byte x (of a 1 KB load, or a row group's rows): the last
// kQStages stages of ring 0, then of ring 1, ...
template <typename C> __device__ inline int q_place(int x) {
  constexpr int PER = C::kQStages * C::kUnit;
  return x / PER * (C::kStages * C::kUnit) + (C::kStages - C::kQStages) * C::kUnit + x % PER;
}

template <typename T, int D, int S, int RG>
__global__ __launch_bounds__(S * RG * 64) void varlen_kernel(const Args a) {
  typedef Shape<D, S, RG> C;
  typedef typename Mma<T>::vec8 V8;
  typedef T T2 __attribute__((ext_vector_type(2)));
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  constexpr int CPR = D / 8, RPL = 64 / CPR, LPW = C::kLpw, NST = C::kStages;
  constexpr int KS = D / 16, DT = D / 32, M = C::kRows;
  // two elements' exponent bits, and what carries all-ones exponents into bit 15
  constexpr uint32_t EXP2 = std::is_same<T, __bf16>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t ONE2 = std::is_same<T, __bf16>::value ? 0x00800080u : 0x04000400u;
  constexpr int GL = 16 / RPL;             // loads of 16 key rows (never more than a page)
  constexpr int GW = LPW < GL ? LPW : GL;  // loads of such a group that a wave makes
  constexpr int NG = LPW / GW;             // groups a wave moves, or shares, per unit
  constexpr bool PIPE = NST >= 4;  // the next unit's scores run under this unit's softmax
  constexpr int STAG = S == 1 && NST >= 8 ? 1 : 0;  // half of the waves a product behind
  static_assert(NG >= 1 && LPW % GW == 0 && GL % GW == 0 && LPW * (NST - 1) < 64 && NST >= 2, "ring");
  extern __shared__ __attribute__((aligned(256))) unsigned char smem[];
  int64_t* table = reinterpret_cast<int64_t*>(smem + C::kRing);  // byte offsets of the chunk's pages in the pool
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + C::kRing + kTableIds * 8);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, lh = lane >> 5;
  const int rg = wave % RG, st = wave / RG;
  const Cut& cut = a.cut;
  const int G = cut.group;

  const int run = run_of_block(blockIdx.x, a.groups);
  if (tid == 0) a.ws_runs[run] = 0;
  LaneSeqs seqs;
  int64_t upto = seqs.load(a.seqs, cut, 0, lane);  // of the chunk in registers
  int64_t total = readlane64(upto, 63);
  if (a.seqs.batch > 64) {
    for (int b0 = 64; b0 < a.seqs.batch; b0 += 64) total += readlane64(seqs.load(a.seqs, cut, b0, lane), 63);
    upto = seqs.load(a.seqs, cut, 0, lane);
  }
  const int64_t per = uniform64(paged::run_length(cut, total, a.groups));
  int64_t at = run * per;  // the run: [at, end) of the line
  if (at >= total) return;
  const int64_t end = at + per < total ? at + per : total;
  int64_t before = 0;  // the line before chunk b0
  while (before + readlane64(upto, 63) <= at) {
    before += readlane64(upto, 63);
    if (seqs.b0 + 64 >= a.seqs.batch) return;  // not reached: at < total
    upto = seqs.load(a.seqs, cut, seqs.b0 + 64, lane);
  }
  int sl = __builtin_ctzll(__ballot(before + upto > at));
  Seq sq = seqs.at(sl);
  Place pl;
  {
    const int64_t start = before + readlane64(upto, sl) - uniform64(paged::head_length(cut, sq)) * cut.num_kv_heads;
    const Place p = paged::place_in_seq(cut, sq, at - start);
    pl.kvh = __builtin_amdgcn_readfirstlane(p.kvh);
    pl.tile = __builtin_amdgcn_readfirstlane(p.tile);
    pl.step = __builtin_amdgcn_readfirstlane(p.step);
    pl.from = uniform64(p.from);
  }
  int64_t left = end - (at - pl.from);  // from the tile's start to the run's end
  // the next sequence with query rows; false behind the last
  auto next_seq = [&]() {
    do {
      if (seqs.b0 + ++sl >= a.seqs.batch) return false;
      if (sl == 64) {
        seqs.load(a.seqs, cut, seqs.b0 + 64, lane);
        sl = 0;
      }
      sq = seqs.at(sl);
    } while (sq.q_len == 0);
    return true;
  };
  if (pl.kvh == cut.num_kv_heads) {
    pl.kvh = 0;
    if (!next_seq()) return;
  }

  // The wave's share of a unit: loads rg LPW .. rg LPW + LPW - 1 of its 4 GL
  // (groups of 16 key rows, 0 and 1 K's, 2 and 3 V's).  Chunk x of row k lies
  // at chunk x ^ swz(k), and both swizzles have a period that divides 16.
  const uint32_t ring = lds_addr(smem) + (uint32_t)(st * NST * C::kUnit);
  constexpr bool BOTH = RG == 1;  // with more row groups a wave moves K or V
  const bool moves_v = !BOTH && rg >= RG / 2;
  uint32_t off[BOTH ? 2 : 1][GW];
#pragma unroll
  for (int i = 0; i < GW; ++i) {
    const int row = (rg * LPW % GL + i) * RPL + lane / CPR;
    const uint32_t at_row = (uint32_t)row * (uint32_t)a.cr * 2u - (uint32_t)i * 1024u;
#pragma unroll
    for (int y = 0; y < (BOTH ? 2 : 1); ++y)
      off[y][i] = at_row + (uint32_t)(((lane % CPR) ^ ((BOTH ? y == 1 : moves_v) ? swz_v<D>(row) : swz_k<D>(row))) << 4);
  }

  for (;;) {
    const int b = seqs.b0 + sl;
    const int n_steps = paged::tile_steps(cut, sq, pl.tile);
    const int s0 = pl.step;
    const int s1 = __builtin_amdgcn_readfirstlane(paged::steps_before(cut, left, n_steps));
    if (s0 >= s1) return;
    const int TG = sq.q_len * G;
    const int r = pl.tile * M + rg * 32 + ln;
    const int R = min(r, TG - 1);
    const int t = (int)fdiv((uint32_t)R, cut.by_group), g = R - t * G;
    const float sl2 = a.scale_log2;

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    // the reference point of the exponentials, where it has to move, it times
    // the scale, the sum
    float m_run = -INFINITY, m_lim = -INFINITY, ms = 0.f, l_run = 0.f;
    const float thr = kRescaleLog2 / sl2;

    const char* hbase = reinterpret_cast<const char*>(static_cast<const T*>(a.cache) + pl.kvh * a.ch);
    const int64_t v_at = a.cs * 2;  // V's bytes behind K's
    const char* wbase = hbase + (moves_v ? v_at : 0);
    const int kl = sq.kv_len, P = sq.prefix;
    const int mask_cols = a.mask != nullptr ? min(min(sq.q_len, a.mask_n), kl - P) : 0;
    // keys that every row of the tile sees: the prefix, or up to the tile's
    // first token's own
    const int seen_by_all = a.mask != nullptr ? P : min(kl, P + (int)fdiv((uint32_t)(pl.tile * M), cut.by_group) + 1);
    const uint8_t* mask_seq = a.mask != nullptr ? a.mask + b * a.mask_seq : nullptr;

    // visibility of keys k0 .. k0 + 31 for token t
    auto word_of = [&](int k0, int tok) {
      if (a.mask == nullptr) {
        const int n = min(max(min(kl, P + tok + 1) - k0, 0), 32);
        return n >= 32 ? 0xffffffffu : (1u << n) - 1u;
      }
      const int np = min(max(P - k0, 0), 32);
      uint32_t w = np >= 32 ? 0xffffffffu : (1u << np) - 1u;
      const int c0 = max(k0 - P, 0);
      if (c0 < mask_cols && k0 + 32 > P && tok < a.mask_n)
        w |= mask_word(mask_seq + tok * a.mask_row, c0, mask_cols) << (c0 + P - k0);
      return w;
    };

    // A tile without keys (kl = 0) has one step that reads nothing.
    int c0 = s0;
    while (c0 < s1 && kl > 0) {
      const int ps = a.seqs.page_shift;
      const paged::Chunk ck = paged::chunk_of(sq, ps, S, c0, s1, a.mask != nullptr);
      const int c1 = ck.end, first_page = ck.first_page, ids = ck.ids, ut0 = ck.tree_unit;
      for (int i = tid; i < ids; i += C::kWaves * 64)
        table[i] = min(max(a.seqs.kv_indices[sq.list + first_page + i], 0), a.seqs.n_pages - 1) * (a.cp * 2);
      barrier();

      // Unit j of the chunk's stream into stage j % NST.  Units that reach past
      // the last key take their rows load by load, each from a block that holds
      // a key, so that no stale value of the pool enters P V.
      const int n = c1 - c0;
      // the pages of the next unit to request, read from the table a step ahead
      int64_t next_page[NG];
      auto peek = [&](int j) {
        const int k0 = ((c0 + j) * S + st) * 32;
#pragma unroll
        for (int x = 0; x < NG; ++x)
          next_page[x] = table[min((min(k0 + 16 * ((rg * LPW / GL + x) & 1), kl - 1) >> ps) - first_page, kTableIds - 1)];
      };
      peek(0);
      auto issue = [&](auto whole_c, int j) {  // whole: the unit ends within the keys
        const int k0 = ((c0 + j) * S + st) * 32;
        const uint32_t dst = ring + (uint32_t)j % NST * C::kUnit;
        if (decltype(whole_c)::value || k0 + 32 <= kl) {
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            const uint32_t row = (uint32_t)(k0 + 16 * ((rg * LPW / GL + x) & 1)) & ((1u << ps) - 1u);
            const bool v_of_both = BOTH && x >= NG / 2;
            const char* base = wbase + (v_of_both ? v_at : 0) + uniform64(next_page[x]) + (uint64_t)row * ((uint32_t)a.cr * 2u);
            dma_rows<GW>(base, off[v_of_both ? 1 : 0], dst + (uint32_t)(rg * LPW + x * GW) * 1024u);
          }
        } else {
          for (int x = 0; x < LPW; ++x) {
            const int u = rg * LPW + x;  // load of the unit
            const bool is_v = u >= 2 * GL;
            const int kb = (u % (2 * GL)) * RPL;
            const int blk = paged::load_block(k0 + kb, RPL, kl);
            const char* base = hbase + (is_v ? v_at : 0) + uniform64(table[(blk >> ps) - first_page]) +
                               (int64_t)(blk & ((1 << ps) - 1)) * a.cr * 2;
            const int row = kb + lane / CPR;
            const int from = min(lane / CPR, kl - 1 - blk);
            const int chunk = (lane % CPR) ^ (is_v ? swz_v<D>(row) : swz_k<D>(row));
            dma_1k(base, (uint32_t)from * (uint32_t)a.cr * 2u + (uint32_t)chunk * 16u, dst + (uint32_t)u * 1024u);
          }
        }
        peek(j + 1);
      };

      i16x8 qf[KS];  // Q^T operand: lane (ln, lh) holds d = 16 kk + 8 lh + [0, 8) of its row
      // S^T of the unit at kt: lane (ln, lh) element i is key 8 (i / 4) + 4 lh
      // + i % 4 of row ln.  K is read KA steps ahead, fenced (left alone, the
      // compiler reads one step ahead and each MFMA waits an LDS latency);
      // between() runs after the first reads, slice(kk) after MFMA kk.
      auto scores = [&](const unsigned char* kt, auto between, auto slice) {
        constexpr int KA = 4;
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        i16x8 kf[KS];
        auto rk = [&](int kk) {
          kf[kk] = *reinterpret_cast<const i16x8*>(kt + ln * C::kRowBytes + (((2 * kk + lh) ^ swz_k<D>(ln)) << 4));
        };
#pragma unroll
        for (int kk = 0; kk < KA; ++kk) rk(kk);
        __builtin_amdgcn_sched_barrier(0);
        between();
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          if (kk + KA < KS) rk(kk + KA);
          s = Mma<T>::run(bit_cast<V8>(kf[kk]), bit_cast<V8>(qf[kk]), s);
          slice(kk);
          __builtin_amdgcn_sched_barrier(0);
        }
        return s;
      };
      auto none = [](auto...) {};
      constexpr std::true_type full{};
      constexpr std::false_type part{};
      int issued = 0;

      // Unit j, whose scores are in s: its row statistics and P (rounded pairs
      // in pk), O re-based where needed.  NEXT: a unit that every row sees
      // whole, unit j + 1's scores (left in s) between its exponentials; else
      // the unit may need its mask (w: the row's visible keys).  STEADY: one
      // unit is due, and it ends within the keys.
      auto soft = [&](auto next_c, auto steady_c, int j, f32x16& s, uint32_t (&pk)[8], uint32_t& w) {
        constexpr bool NEXT = decltype(next_c)::value, STEADY = decltype(steady_c)::value;
        const int u = (c0 + j) * S + st;
        auto stats = [&]() {
          if (!NEXT && (u + 1) * 32 > seen_by_all) {
            w = a.mask != nullptr ? words[(u - ut0) * M + rg * 32 + ln] : word_of(u * 32, t);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!((w >> (8 * (i >> 2) + 4 * lh + (i & 3))) & 1u)) s[i] = -INFINITY;
          }
          const float mx = max16f<!NEXT>(s);
          const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          const float rmax = max3f(__uint_as_float(sw[0]), __uint_as_float(sw[1]), __uint_as_float(sw[1]));
          // the reference point moves only when a score passes it by more than
          // 2^8 (exact for any consistent point; p stays below 2^8)
          const bool need = rmax > m_lim;
          if (__ballot(need) != 0) {
            const float m_new = need ? rmax : m_run;
            const float alpha = need ? __builtin_amdgcn_exp2f((m_run - m_new) * sl2) : 1.f;
            m_run = m_new;
            m_lim = m_new + thr;
            ms = m_new == -INFINITY ? 0.f : m_new * sl2;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
          }
        };
        // P is rounded to the input type for the product with V, which takes
        // 16-bit operands; its row sum takes the unrounded values.  Pinned where
        // they are computed: the compiler sinks them past the re-base otherwise.
        float psum = 0.f, p[16];
        auto expo = [&](int i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sl2, -ms));
          psum += p[i];
          if (i & 1) {
            pk[i >> 1] = bit_cast<uint32_t>(T2{(T)p[i - 1], (T)p[i]});
            asm volatile("" : "+v"(pk[i >> 1]), "+v"(psum));
          }
        };
        if constexpr (NEXT) {
          const f32x16 sn = scores(smem + (st * NST + (uint32_t)(j + 1) % NST) * C::kUnit, [&]() {
            if constexpr (STEADY) issue(full, issued++);
            else while (issued < min(n, j + NST - STAG)) issue(part, issued++);
            stats();
          }, [&](int kk) {
#pragma unroll
            for (int i = 16 / KS * kk; i < 16 / KS * (kk + 1); ++i) expo(i);
          });
          s = sn;
        } else {
          stats();
#pragma unroll
          for (int i = 0; i < 16; ++i) expo(i);
        }
        l_run += psum;
      };

      // O^T += V^T P^T of unit j.  V^T by the transposing LDS read: lane i of
      // 16-lane group x gets keys 16 s2 + 8 jj + 4 (x >> 1) + [0, 4) of
      // d = 32 dt + 16 (x & 1) + i, the key order in which P lies; products of
      // one d tile lie DT apart.
      auto pv = [&](auto next_c, int j, const uint32_t (&pk)[8], uint32_t w) {
        constexpr bool NEXT = decltype(next_c)::value;
        const unsigned char* vt = smem + (st * NST + (uint32_t)j % NST) * C::kUnit + C::kTile;
        const V8 pb[2] = {bit_cast<V8>(U4{pk[0], pk[1], pk[2], pk[3]}), bit_cast<V8>(U4{pk[4], pk[5], pk[6], pk[7]})};
        const int vx = lane >> 4, vi = lane & 15;
        const int vrow = 4 * (vx >> 1) + (vi >> 2);
        const int vch = 2 * (vx & 1) + ((vi & 3) >> 1), vhalf = 8 * (vi & 1);
        const uint32_t vb = lds_addr(vt) + (uint32_t)(vrow * C::kRowBytes + ((vch ^ swz_v<D>(vrow)) << 4) + vhalf);
        i16x4 vh[2 * DT][2];
        auto rv = [&](int x) {  // x = s2 DT + dt: dt moves offset bits 6 and 7 under the XOR
          const TSFA_LDS char* at = (const TSFA_LDS char*)(uintptr_t)(vb ^ (uint32_t)((x % DT) << 6));
          vh[x][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TSFA_LDS i16x4*)(at + 16 * (x / DT) * C::kRowBytes));
          vh[x][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TSFA_LDS i16x4*)(at + (16 * (x / DT) + 8) * C::kRowBytes));
        };
        bool odd = false;
        if (!NEXT && ((c0 + j) * S + st + 1) * 32 > seen_by_all) {
          // infinities and NaN of keys that some rows do not see: 0 * NaN must
          // not reach those rows, so they leave the product and are added to
          // the rows that see them
          uint32_t hit = 0;
#pragma unroll
          for (int i = 0; i < C::kTile / 1024; ++i) {
            const U4 v4 = *reinterpret_cast<const U4*>(vt + 1024 * i + 16 * lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) hit |= ((v4[e] & EXP2) + ONE2) & 0x80008000u;
          }
          odd = __ballot(hit != 0) != 0;
        }
        constexpr int VA = 3;
#pragma unroll
        for (int x = 0; x < VA; ++x) rv(x);
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x) {
          if (x + VA < 2 * DT) rv(x + VA);
          i16x8 f = __builtin_shufflevector(vh[x][0], vh[x][1], 0, 1, 2, 3, 4, 5, 6, 7);
          if (!NEXT && odd) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if ((f[e] & (short)(EXP2 & 0xffff)) == (short)(EXP2 & 0xffff)) f[e] = 0;
          }
          o[x % DT] = Mma<T>::run(bit_cast<V8>(f), pb[x / DT], o[x % DT]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!NEXT && odd) {
#pragma unroll 1
          for (int key = 0; key < 32; ++key) {
            const bool seen = (w >> key) & 1u;
            const unsigned char* row = vt + key * C::kRowBytes + 8 * lh;
#pragma unroll
            for (int x = 0; x < D / 8; ++x) {
              const T4 v = *reinterpret_cast<const T4*>(row + ((x ^ swz_v<D>(key)) << 4));
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float f = (float)v[e];
                o[x >> 2][4 * (x & 3) + e] += seen && !(f - f == 0.f) ? f : 0.f;
              }
            }
          }
        }
      };

      vm_wait<0>();  // the ring's waits count its own loads and Q's alone
      // Q comes through the rings' last stages, rows whole, in K's layout (16
      // bytes a lane straight from the rows touch a cache line per lane: 2 us
      // of a tile's start).
#pragma unroll 1
      for (int i = 0; i < C::kQLoads; ++i) {
        const int row = (wave * C::kQLoads + i) * RPL + lane / CPR;
        const int rr = min(pl.tile * M + row, TG - 1);
        const int tt = (int)fdiv((uint32_t)rr, cut.by_group), gg = rr - tt * G;
        const T* src = static_cast<const T*>(a.q) + (int64_t)(sq.q0 + tt) * a.sqn + (int64_t)(pl.kvh * G + gg) * a.sqh +
                       (((lane % CPR) ^ swz_k<D>(row)) << 3);
        dma_1k_rows(src, lds_addr(smem) + q_place<C>((wave * C::kQLoads + i) * 1024));
      }
      while (issued < C::kAhead && issued < n) issue(part, issued++);
      if (a.mask != nullptr) {
        // under the first units' way here; the barriers below order them
        for (int i = tid; i < (c1 * S - ut0) * M; i += C::kWaves * 64) {
          const int row = min(pl.tile * M + i % M, TG - 1);
          words[i] = word_of((ut0 + i / M) * 32, (int)fdiv((uint32_t)row, cut.by_group));
        }
      }
      int j = 0;
      wait_units<LPW, NST - 2>(issued - 1);
      barrier();
      {
        const unsigned char* qt = smem + q_place<C>(rg * 32 * C::kRowBytes) + ln * C::kRowBytes;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
          qf[kk] = *reinterpret_cast<const i16x8*>(qt + (((2 * kk + lh) ^ swz_k<D>(ln)) << 4)) ^
                   (short)(a.neg_q ? 0x8000 : 0);
      }
      if constexpr (RG == 1) barrier();  // below, a stream's ring and steps are its wave's own
      // unit 1 takes Q's stage: it has to be on its way before step 1 waits
      static_assert(C::kAhead >= 2 || RG == 1, "Q is read");
      if constexpr (C::kAhead < 2)
        while (issued < min(n, NST)) issue(part, issued++);
      f32x16 s = scores(smem + st * NST * C::kUnit, none, none);
      uint32_t pk[8], w = 0xffffffffu;
      if constexpr (PIPE) {
        // Steps whose units every row of the tile sees whole.  Past barrier j
        // unit j + 1 is there, and every wave is done with unit j - 1 (with
        // STAG, j - 2).  With STAG half of the waves meet at barrier j + 1
        // before the product of unit j: the other wave of their SIMD is then at
        // its exponentials while they run it, and the other way round.
        const int n_full = min(n, seen_by_all / (32 * S) - c0);
        const bool late = STAG != 0 && rg >= RG / 2;
        auto meet = [&](auto steady_c, int i) {
          if (decltype(steady_c)::value) vm_wait<(NST - 3 - STAG) * LPW>();  // issued = i + NST - 1 - STAG
          else wait_units<LPW, NST - 3>(issued - 2 - i);
          stream_barrier<RG == 1>();
        };
        auto step = [&](auto steady_c) {
          if (!late) meet(steady_c, j);
          soft(full, steady_c, j, s, pk, w);
          if (late && (decltype(steady_c)::value || j + 2 < n_full)) meet(steady_c, j + 1);
          pv(full, j, pk, w);
          ++j;
        };
        // Steady from step 1 on, while every step requests one unit that ends
        // within the keys: what is on its way is a constant then.
        const int n_steady = min(n_full - 2, min(n, kl / (32 * S) - c0) - (NST - 1 - STAG));
        if (late && n_full > 1) meet(part, 0);
        while (j + 1 < n_full) {
          step(part);
          while (j < n_steady) step(full);
        }
      }
      for (;;) {
        w = 0xffffffffu;
        soft(part, part, j, s, pk, w);
        pv(part, j, pk, w);
        if (++j >= n) break;
        wait_units<LPW, NST - 2>(issued - 1 - j);
        stream_barrier<RG == 1>();  // unit j is there, and every wave is done with unit j - 1
        while (issued < min(n, j + NST)) issue(part, issued++);
        s = scores(smem + (st * NST + (uint32_t)j % NST) * C::kUnit, none, none);
      }
      barrier();  // the rings, the table and the words are free again
      c0 = c1;
    }
    l_run += __shfl_xor(l_run, 32);

    // The streams' results join in LDS, every wave finishing 1 / S of its row
    // group's columns: a lane's float4 x holds d = 8 x + 4 lh .. + 3, stream s
    // takes x in [s X / S, (s + 1) X / S).
    constexpr int X = D / 8, XS = X / S;
    const bool whole = s0 == 0 && s1 == n_steps;
    float4* jo = reinterpret_cast<float4*>(smem);                              // the streams' O
    float2* jml = reinterpret_cast<float2*>(smem + C::kRing + kTableIds * 8);  // [S][RG][32] (m, l)
    static_assert(S * RG * 32 * 8 <= C::kWords && (S == 1 || S * RG * X * 1024 <= C::kRing), "join");
    if (S > 1 && lh == 0) jml[(st * RG + rg) * 32 + ln] = make_float2(m_run, l_run);
    float mm = -INFINITY, ll = 0.f, fs[S];
    auto weights = [&]() {
      float2 ml[S];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        ml[i] = jml[(i * RG + rg) * 32 + ln];
        mm = fmaxf(mm, ml[i].x);
      }
      const float m0 = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        fs[i] = __builtin_amdgcn_exp2f((ml[i].x - m0) * sl2);
        ll += ml[i].y * fs[i];
      }
    };
    // a tile of one run: O; a shared one: slot 2 run if it began before the
    // run, else 2 run + 1
    T* orow = static_cast<T*>(a.out) + (int64_t)(sq.q0 + t) * a.son + (int64_t)(pl.kvh * G + g) * a.soh + 4 * lh;
    const int64_t slot = 2 * (int64_t)run + (s0 == 0 ? 1 : 0);
    float4* wo = a.ws_o + (slot * RG + rg) * X * 64 + lane;
    auto put = [&](int x, float4 v) {
      if (whole) {
        const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);  // NaN stays
        const T4 r4 = {(T)(v.x * inv), (T)(v.y * inv), (T)(v.z * inv), (T)(v.w * inv)};
        if (r < TG) *reinterpret_cast<T4*>(orow + 8 * x) = r4;
      } else {
        wo[x * 64] = v;
      }
    };
    auto o4 = [&](int x) {
      const int dt = x >> 2, i = x & 3;
      return make_float4(o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]);
    };
    if constexpr (S == 1) {
      mm = m_run;
      ll = l_run;
#pragma unroll
      for (int x = 0; x < X; ++x) put(x, o4(x));
    } else if constexpr (S == 2) {
      // each stream leaves the other's half and finishes its own
      float4* mine = jo + ((st * RG + rg) * XS) * 64 + lane;
      const float4* other = jo + (((1 - st) * RG + rg) * XS) * 64 + lane;
      auto half = [&](auto st_c) {
        constexpr int ST = decltype(st_c)::value;
#pragma unroll
        for (int x = 0; x < XS; ++x) mine[x * 64] = o4((1 - ST) * XS + x);
        barrier();
        weights();
#pragma unroll
        for (int x = 0; x < XS; ++x) {
          const float4 u = o4(ST * XS + x), v = other[x * 64];
          put(ST * XS + x, make_float4(u.x * fs[ST] + v.x * fs[1 - ST], u.y * fs[ST] + v.y * fs[1 - ST],
                                       u.z * fs[ST] + v.z * fs[1 - ST], u.w * fs[ST] + v.w * fs[1 - ST]));
        }
      };
      if (st == 0) half(std::integral_constant<int, 0>{});
      else half(std::integral_constant<int, 1>{});
    } else {
#pragma unroll
      for (int x = 0; x < X; ++x) jo[((st * RG + rg) * X + x) * 64 + lane] = o4(x);
      barrier();
      weights();
#pragma unroll
      for (int y = 0; y < XS; ++y) {
        const int x = st * XS + y;
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const float4 v = jo[((i * RG + rg) * X + x) * 64 + lane];
          u.x += v.x * fs[i];
          u.y += v.y * fs[i];
          u.z += v.z * fs[i];
          u.w += v.w * fs[i];
        }
        put(x, u);
      }
    }
    if (st == 0 && lh == 0) {
      if (!whole) {
        a.ws_ml[slot * M + rg * 32 + ln] = make_float2(mm, ll);
      } else if (a.lse != nullptr && r < TG) {
        a.lse[(int64_t)(sq.q0 + t) * a.num_heads + pl.kvh * G + g] =
            ll == 0.f ? -INFINITY : mm * (sl2 * 0.6931471805599453f) + logf(ll);
      }
    }
    if (tid == 0 && s0 == 0 && s1 < n_steps) {
      const int64_t tile_at = end - left;  // the run that the tile's last step starts in:
      const int64_t last = paged::udiv(tile_at + (n_steps - 1) * cut.unit, per, paged::inverse(per));
      a.ws_runs[run] = (int)(last - run) + 1;
      a.ws_desc[run] = Args::Desc{sq.q0, sq.q_len, pl.kvh, pl.tile, tile_at, per};
    }

    // on along the line
    if (s1 < n_steps) return;
    barrier();  // the ring is written again
    left -= paged::tile_first(cut, sq) + paged::tile_more(cut) * pl.tile;
    if (left <= 0) return;
    pl.step = 0;
    if (++pl.tile == paged::cut_tiles(cut, sq)) {
      pl.tile = 0;
      if (++pl.kvh == cut.num_kv_heads) {
        pl.kvh = 0;
        if (!next_seq()) return;
      }
    }
  }
}

// Joins the parts of the tiles that several runs share.  Work items are (tile,
// row group, d tile); every block lists the tiles first (one load of all runs'
// descriptors).  Tiles of up to kJoin parts take a wave per item, longer ones a
// block whose four waves split the parts, kJoin of them loaded at once.  (A
// block per run would leave most of them empty and the others few: 17 us against
// 6 for 16 tiles in 14 parts each.)
constexpr int kJoin = 4;
constexpr int kMaxGroups = 1024;  // a run's number takes 10 bits

// Parts p0, p0 + step, ... of a lane's row and d tile, joined into (m, l, o).
template <int D, int RG>
__device__ inline void join_parts(const Args& a, const Args::Desc& desc, int run, int runs, int rg, int dt, int p0,
                                  int step, int lane, float& m, float& l, float4 (&o)[4]) {
  constexpr int M = 32 * RG;
  const float sl2 = a.scale_log2;
  for (; p0 < runs; p0 += step * kJoin) {
    float2 x[kJoin];
    float4 v[kJoin][4];
    bool has[kJoin];
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      // past the last and runs without a step of the tile: loaded, not used
      const int p = min(p0 + step * k, runs - 1);
      has[k] = p0 + step * k < runs && paged::run_has_step(a.cut, (int64_t)(run + p) * desc.per, desc.per, desc.at);
      const int64_t slot = p == 0 ? 2 * (int64_t)run + 1 : 2 * (int64_t)(run + p);
      x[k] = a.ws_ml[slot * M + rg * 32 + (lane & 31)];
      const float4* wo = a.ws_o + ((slot * RG + rg) * (D / 8) + 4 * dt) * 64 + lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] = wo[i * 64];
      if (!has[k]) x[k] = make_float2(-INFINITY, 0.f);
    }
    float m_new = m;
#pragma unroll
    for (int k = 0; k < kJoin; ++k) m_new = fmaxf(m_new, x[k].x);
    const float m0 = m_new == -INFINITY ? 0.f : m_new;
    const float fa = __builtin_amdgcn_exp2f((m - m0) * sl2);
    m = m_new;
    l *= fa;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float4(o[i].x * fa, o[i].y * fa, o[i].z * fa, o[i].w * fa);
#pragma unroll
    for (int k = 0; k < kJoin; ++k) {
      if (!has[k]) continue;
      const float f = __builtin_amdgcn_exp2f((x[k].x - m0) * sl2);
      l += x[k].y * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i].x += v[k][i].x * f;
        o[i].y += v[k][i].y * f;
        o[i].z += v[k][i].z * f;
        o[i].w += v[k][i].w * f;
      }
    }
  }
}

template <typename T, int D, int RG>
__global__ __launch_bounds__(256) void combine_kernel(const Args a) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int DT = D / 32, PS = 4, M = 32 * RG;
  __shared__ float4 jo[PS * 4 * 64];
  __shared__ float2 jml[PS * 64];
  __shared__ int tiles[kMaxGroups];  // run and, above, how many it goes on for
  __shared__ int wave_count[kMaxGroups / 64];
  __shared__ int any_long;
  const int lane = threadIdx.x & 63, ps = threadIdx.x >> 6;
  const int ln = lane & 31, lh = lane >> 5;
  if (threadIdx.x == 0) any_long = 0;
  __syncthreads();
  for (int r0 = ps * 64; r0 < a.groups; r0 += 256) {
    const int runs = r0 + lane < a.groups ? a.ws_runs[r0 + lane] : 0;
    const uint64_t set = __ballot(runs != 0);
    if (lane == 0) wave_count[r0 / 64] = __builtin_popcountll(set);
    if (runs > kJoin) any_long = 1;
  }
  __syncthreads();
  int n_tiles = 0;
  for (int w = 0; w * 64 < a.groups; ++w) n_tiles += wave_count[w];
  const int n_items = n_tiles * RG * DT;
  if ((int)blockIdx.x >= n_items) return;
  for (int r0 = ps * 64; r0 < a.groups; r0 += 256) {
    const int runs = r0 + lane < a.groups ? a.ws_runs[r0 + lane] : 0;
    int at = __builtin_popcountll(__ballot(runs != 0) & ((1ull << lane) - 1));
    for (int w = 0; w < r0 / 64; ++w) at += wave_count[w];
    if (runs != 0) tiles[at] = (runs << 10) | (r0 + lane);
  }
  __syncthreads();
  const float sl2 = a.scale_log2;
  // float4 x of the lane's row and d tile: normalised, rounded and written
  auto put = [&](const Args::Desc& desc, int rg, int dt, int x, float4 r, float m, float l) {
    const int G = a.cut.group, row = desc.tile * M + rg * 32 + ln;
    if (row >= desc.q_len * G) return;
    const int t = (int)fdiv((uint32_t)row, a.cut.by_group), h = desc.kvh * G + (row - t * G);
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const T4 v = {(T)(r.x * inv), (T)(r.y * inv), (T)(r.z * inv), (T)(r.w * inv)};
    *reinterpret_cast<T4*>(static_cast<T*>(a.out) + (int64_t)(desc.q0 + t) * a.son + (int64_t)h * a.soh + 32 * dt +
                           8 * x + 4 * lh) = v;
    if (a.lse != nullptr && dt == 0 && x == 0 && lh == 0)
      a.lse[(int64_t)(desc.q0 + t) * a.num_heads + h] =
          l == 0.f ? -INFINITY : m * (sl2 * 0.6931471805599453f) + logf(l);
  };
  for (int item = blockIdx.x * PS + ps; item < n_items; item += gridDim.x * PS) {
    const int tile = __builtin_amdgcn_readfirstlane(tiles[item / (RG * DT)]);
    const int run = tile & (kMaxGroups - 1), runs = tile >> 10, rg = item / DT % RG, dt = item % DT;
    const Args::Desc desc = a.ws_desc[run];
    if (runs > kJoin || desc.tile * M + rg * 32 >= desc.q_len * a.cut.group) continue;
    float m = -INFINITY, l = 0.f;
    float4 o[4] = {};
    join_parts<D, RG>(a, desc, run, runs, rg, dt, 0, 1, lane, m, l, o);
#pragma unroll
    for (int x = 0; x < 4; ++x) put(desc, rg, dt, x, o[x], m, l);
  }
  if (any_long == 0) return;
  for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
    const int tile = __builtin_amdgcn_readfirstlane(tiles[item / (RG * DT)]);
    const int run = tile & (kMaxGroups - 1), runs = tile >> 10, rg = item / DT % RG, dt = item % DT;
    const Args::Desc desc = a.ws_desc[run];
    if (runs <= kJoin || desc.tile * M + rg * 32 >= desc.q_len * a.cut.group) continue;
    float m = -INFINITY, l = 0.f;
    float4 o[4] = {};
    join_parts<D, RG>(a, desc, run, runs, rg, dt, ps, PS, lane, m, l, o);
    jml[ps * 64 + lane] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) jo[(ps * 4 + i) * 64 + lane] = o[i];
    __syncthreads();
    // wave ps takes the lane's float4 ps
    m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PS; ++k) m = fmaxf(m, jml[k * 64 + lane].x);
    const float m0 = m == -INFINITY ? 0.f : m;
    l = 0.f;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PS; ++k) {
      const float2 ml = jml[k * 64 + lane];
      const float f = __builtin_amdgcn_exp2f((ml.x - m0) * sl2);
      const float4 v = jo[(k * 4 + ps) * 64 + lane];
      l += ml.y * f;
      r.x += v.x * f;
      r.y += v.y * f;
      r.z += v.z * f;
      r.w += v.w * f;
    }
    put(desc, rg, dt, ps, r, m, l);
    __syncthreads();  // jo and jml are written again
  }
}

struct Sizes {
  int groups, rows, streams, extra;
  size_t o, ml, runs, desc;
  size_t total() const { return o + ml + runs + desc; }
};

// Rows of a tile, by the rows of a sequence (query token x head of a kv head)
// and by the work: the steps of 128 rows x 64 keys that a workgroup would take,
// sequences and lists (`keys` of them to a sequence) at their mean.
// 32 rows and four key streams for sequences of up to 32 rows, and where there
// is little work, for such a tile starts and ends sooner: up to 5 steps, or 32
// where two tiles of 32 rows read the keys as often as one of 128 (and while the
// tiles are few: a run that holds pieces of three loses that again).
// 128 rows and two streams above.  Time with 128 rows over time with 32, D 128,
// at 2, 4, 5 and 6 steps: 96 rows a sequence 1.22 1.01 0.92 0.89, 128 rows 1.27
// 1.09 1.05 1.03, 192 rows 1.12 1.01 0.97 0.93, 256 rows 1.25 1.17 1.11 1.04, D 64
// 1.00 to 1.20 at all of these; 64 rows at 8, 16, 32 and 64 steps 1.18 1.09 0.99
// 0.93, D 64 1.30 1.27 1.18 1.02.
// 256 rows and one stream where there is much work, for it reads the keys half
// as often: 512 to 2048 rows of 16 sequences by 4096 keys (132 steps and more)
// 160 to 675 us against 184 to 803 us with 128 rows, 8 x 1024 rows by 2300 (72
// steps) 100 against 113, 8 x 512 rows by 2176 (34 steps) 62 against 57, 2048 rows
// by 4600 (36 steps) 69 against 65.
constexpr double kLittleWork = 5, kLittleWork64 = 32, kMuchWork = 64;  // steps
constexpr int64_t kMaxKeys = 1 << 30;
inline Sizes sizes_of(int cus, int batch, int total_q, int num_heads, int num_kv_heads, int head_dim, int64_t keys) {
  Sizes s;
  s.groups = cus < kMaxGroups ? cus : kMaxGroups;
  const int64_t rows = (int64_t)total_q * (num_heads / num_kv_heads);  // <= 2^30
  // tiles of n rows
  auto tiles = [&](int64_t n) { return (rows + n * batch - 1) / (n * batch) * batch * num_kv_heads; };
  const double steps = (double)tiles(128) * (double)(keys < kMaxKeys ? keys : kMaxKeys) / (64.0 * s.groups);
  const bool little = tiles(32) <= s.groups * 3 / 4 &&
                      steps <= (rows <= (int64_t)64 * batch ? kLittleWork64 : kLittleWork);
  s.rows = rows <= (int64_t)32 * batch || little ? 32 : rows > (int64_t)256 * batch && steps >= kMuchWork ? 256 : 128;
  s.streams = s.rows == 32 ? 4 : s.rows == 256 ? 1 : 2;
  s.extra = s.rows == 32 ? 2 : 8;
  s.o = align256((size_t)2 * s.groups * s.rows * head_dim * 4);
  s.ml = align256((size_t)2 * s.groups * s.rows * 8);
  s.runs = align256((size_t)s.groups * 4);
  s.desc = align256((size_t)s.groups * sizeof(Args::Desc));
  return s;
}

int check(int batch, int total_q, int num_heads, int num_kv_heads, int head_dim, int dtype) {
  if (batch < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return TSFA_ERR_INVALID_ARGUMENT;
  if (dtype != TSFA_DTYPE_FP16 && dtype != TSFA_DTYPE_BF16) return TSFA_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return TSFA_ERR_UNSUPPORTED;
  if (num_heads / num_kv_heads > 256 || (int64_t)total_q * (num_heads / num_kv_heads) > (1 << 30))
    return TSFA_ERR_UNSUPPORTED;
  return TSFA_OK;
}

template <typename T, int D, int S, int RG> int launch(const Args& a, hipStream_t s) {
  typedef Shape<D, S, RG> C;
  static_assert(C::kLds <= 163840, "LDS");
  // the LDS limit attribute is set once per device
  static std::atomic<uint64_t> attr_set{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return TSFA_ERR_DEVICE;
  const uint64_t bit = 1ull << (dev & 63);
  if ((attr_set.load(std::memory_order_acquire) & bit) == 0) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&varlen_kernel<T, D, S, RG>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds) != hipSuccess)
      return TSFA_ERR_LAUNCH;
    attr_set.fetch_or(bit, std::memory_order_acq_rel);
  }
  hipLaunchKernelGGL((varlen_kernel<T, D, S, RG>), dim3((unsigned)a.groups), dim3(C::kWaves * 64), C::kLds, s, a);
  hipLaunchKernelGGL((combine_kernel<T, D, RG>), dim3((unsigned)a.groups * 4), dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? TSFA_OK : TSFA_ERR_LAUNCH;
}

template <typename T, int D> int launch_tiles(const Args& a, int rows, hipStream_t s) {
  if (rows == 32) return launch<T, D, 4, 1>(a, s);
  return rows == 128 ? launch<T, D, 2, 4>(a, s) : launch<T, D, 1, 8>(a, s);
}

}  // namespace varlen
}  // namespace tsfa

using namespace tsfa;

extern "C" size_t tsfa_fwd_paged_varlen_workspace_bytes(int batch, int total_q, int num_heads, int num_kv_heads,
                                                        int head_dim, int dtype) {
  int cus = 0;
  if (varlen::check(batch, total_q, num_heads, num_kv_heads, head_dim, dtype) != TSFA_OK || batch == 0 || total_q == 0)
    return 0;
  if (device_cu_count(&cus) != TSFA_OK) return 0;
  // the larger of the tiles a call with these rows may take
  return varlen::sizes_of(cus, batch, total_q, num_heads, num_kv_heads, head_dim, varlen::kMaxKeys).total();
}

extern "C" int tsfa_fwd_paged_varlen(const void* q, const void* kv_cache, void* o, float* lse, const uint8_t* mask,
                                     int64_t mask_seq_stride, int64_t mask_row_stride, int mask_n,
                                     const int32_t* q_indptr, const int32_t* kv_lens, const int32_t* kv_indptr,
                                     const int32_t* kv_indices, int64_t n_indices, int64_t page_table_stride,
                                     int page_table_width, int n_pages, int page_size, const int64_t* q_strides,
                                     const int64_t* cache_strides, const int64_t* o_strides, float sm_scale, int batch,
                                     int total_q, int num_heads, int num_kv_heads, int head_dim, int dtype,
                                     void* workspace, size_t workspace_bytes, tsfa_stream_t stream) {
  int st = varlen::check(batch, total_q, num_heads, num_kv_heads, head_dim, dtype);
  if (st != TSFA_OK) return st;
  if (q_strides == nullptr || cache_strides == nullptr || o_strides == nullptr || !(sm_scale - sm_scale == 0.f))
    return TSFA_ERR_INVALID_ARGUMENT;
  if (mask != nullptr && (mask_n <= 0 || mask_seq_stride < 0 || mask_row_stride < 0)) return TSFA_ERR_INVALID_ARGUMENT;
  st = paged_check(kv_indptr, n_indices, page_table_stride, page_table_width, n_pages, page_size, batch);
  if (st != TSFA_OK) return st;
  for (const int64_t* p : {q_strides, o_strides})
    if (p[2] != 1 || p[0] % 8 != 0 || p[1] % 8 != 0) return TSFA_ERR_UNSUPPORTED;
  for (int i = 0; i < 4; ++i)
    if (cache_strides[i] % 8 != 0) return TSFA_ERR_UNSUPPORTED;
  // a lane's offset from its load's first row is an unsigned 32-bit byte count
  if (cache_strides[4] != 1 || cache_strides[2] < head_dim || cache_strides[2] > ((int64_t)1 << 26))
    return TSFA_ERR_UNSUPPORTED;
  if (batch == 0 || total_q == 0) return TSFA_OK;
  for (const void* p : {q, kv_cache, (const void*)o}) {
    if (p == nullptr) return TSFA_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return TSFA_ERR_UNSUPPORTED;
  }
  if (q_indptr == nullptr || kv_lens == nullptr || (kv_indices == nullptr && n_indices > 0))
    return TSFA_ERR_INVALID_ARGUMENT;
  int cus = 0;
  if (device_cu_count(&cus) != TSFA_OK) return TSFA_ERR_DEVICE;
  const int64_t keys = (kv_indptr != nullptr ? n_indices / batch : (int64_t)page_table_width) * page_size;
  const varlen::Sizes sz = varlen::sizes_of(cus, batch, total_q, num_heads, num_kv_heads, head_dim, keys);
  if (workspace == nullptr || workspace_bytes < sz.total() || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return TSFA_ERR_WORKSPACE;

  varlen::Args a;
  a.q = q;
  a.cache = kv_cache;
  a.out = o;
  a.lse = lse;
  a.mask = mask;
  a.mask_seq = mask_seq_stride;
  a.mask_row = mask_row_stride;
  a.mask_n = mask_n;
  a.seqs = make_seqs(q_indptr, kv_lens, kv_indptr, kv_indices, n_indices, page_table_stride, page_table_width, n_pages,
                     page_size, batch, total_q);
  a.cut = paged::make_cut(sz.rows, 32 * sz.streams, num_heads / num_kv_heads, num_kv_heads, mask == nullptr, sz.extra);
  a.sqn = q_strides[0], a.sqh = q_strides[1];
  a.son = o_strides[0], a.soh = o_strides[1];
  a.cp = cache_strides[0], a.cs = cache_strides[1], a.cr = cache_strides[2], a.ch = cache_strides[3];
  const float sl2 = fabsf(sm_scale) * 1.4426950408889634f;
  a.scale_log2 = sl2 > 1e-30f ? sl2 : 1e-30f;  // 0: every score weighs the same, masked ones stay -inf
  a.neg_q = sm_scale < 0.f;
  a.num_heads = num_heads;
  a.groups = sz.groups;
  char* ws = static_cast<char*>(workspace);
  a.ws_o = reinterpret_cast<float4*>(ws);
  a.ws_ml = reinterpret_cast<float2*>(ws + sz.o);
  a.ws_runs = reinterpret_cast<int*>(ws + sz.o + sz.ml);
  a.ws_desc = reinterpret_cast<varlen::Args::Desc*>(ws + sz.o + sz.ml + sz.runs);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TSFA_DTYPE_BF16)
    return head_dim == 128 ? varlen::launch_tiles<__bf16, 128>(a, sz.rows, s) : varlen::launch_tiles<__bf16, 64>(a, sz.rows, s);
  return head_dim == 128 ? varlen::launch_tiles<_Float16, 128>(a, sz.rows, s)
                         : varlen::launch_tiles<_Float16, 64>(a, sz.rows, s);
}
