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
// are S key streams of RG row groups of 32 rows: S = 2, RG = 4 for trees
// (128 rows share each key), S = 4, RG = 1 where a sequence has 32 rows or
// fewer (decoding: every wave streams keys of its own).  A step is 32 S keys;
// stream s takes 32 of them through its own LDS ring (global_load_lds, HBM ->
// LDS without registers).  S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16: a lane holds one query row in both, so the softmax
// statistics stay in the lane, with one exchange between the lane halves.
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
  int4* ws_desc;                   // [groups] the tile that starts in the run and ends behind it
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
#pragma clang diagnostic pop
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

// The place of the line's step `at`, and the line's length in *total; every
// lane of a wave calls it and gets the same answer.  Lanes take 64 sequences
// at a time.
__device__ inline int64_t lane_scan(int64_t x, int lane) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int64_t y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  return x;
}
__device__ inline int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
struct Line {
  int64_t total, per;  // steps in all, steps of one workgroup
  int used;            // workgroups with work
};
__device__ inline Line line_of(const paged::Seqs& s, const Cut& c, int groups, int lane) {
  int64_t sum = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    const int b = b0 + lane;
    int64_t x = b < s.batch ? paged::head_steps(c, paged::seq_of(s, b)) * c.num_kv_heads : 0;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    sum += uniform64(x);
  }
  Line l;
  l.total = sum;
  l.per = (sum + groups - 1) / groups;
  l.used = sum > 0 ? (int)((sum + l.per - 1) / l.per) : 0;
  return l;
}
__device__ inline Place place_at(const paged::Seqs& s, const Cut& c, int64_t at, int lane) {
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    const int b = b0 + lane;
    const int64_t mine = b < s.batch ? paged::head_steps(c, paged::seq_of(s, b)) * c.num_kv_heads : 0;
    const int64_t upto = lane_scan(mine, lane);
    const uint64_t past = __ballot(upto > at);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      const int64_t before = uniform64(__shfl(upto - mine, l));
      const int bb = __builtin_amdgcn_readfirstlane(b0 + l);
      return paged::place_in_seq(c, paged::seq_of(s, bb), bb, at - before);
    }
    at -= uniform64(__shfl(upto, 63));
  }
  Place none;
  none.b = -1;  // not reached with at < total
  return none;
}

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
  static constexpr int kLds = kRing + kTableIds * 4 + kWords;
};

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
  static_assert(LPW >= 1 && LPW * (NST - 1) < 64 && NST >= 2, "ring");
  extern __shared__ __attribute__((aligned(256))) unsigned char smem[];
  int32_t* table = reinterpret_cast<int32_t*>(smem + C::kRing);
  uint32_t* words = reinterpret_cast<uint32_t*>(smem + C::kRing + kTableIds * 4);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, lh = lane >> 5;
  const int rg = wave % RG, st = wave / RG;
  const Cut& cut = a.cut;
  const int G = cut.group;

  const int run = run_of_block(blockIdx.x, a.groups);
  const Line line = line_of(a.seqs, cut, a.groups, lane);
  if (tid == 0) a.ws_desc[run] = make_int4(0, 0, 0, 0);
  if (run >= line.used) return;
  int64_t at = run * line.per;
  const int64_t end = at + line.per < line.total ? at + line.per : line.total;
  Place pl = place_at(a.seqs, cut, at, lane);
  if (pl.b < 0) return;

  // the wave's share of a unit: rows [row0, row0 + rows) of K or V
  constexpr int HALF = LPW * RG / 2;  // loads of one tile
  const uint32_t ring = lds_addr(smem) + (uint32_t)(st * NST * C::kUnit);

  for (;;) {
    const int b = pl.b;
    const Seq sq = pl.seq;
    const int n_steps = paged::tile_steps(cut, sq, pl.tile);
    const int s0 = pl.step;
    const int s1 = (int)(end - at < n_steps - s0 ? s0 + (end - at) : n_steps);
    const int TG = sq.q_len * G;
    const int r = pl.tile * M + rg * 32 + ln;
    const int R = min(r, TG - 1);
    const int t = R / G, g = R - t * G;
    const float sl2 = a.scale_log2;

    // Q^T operand: lane (ln, lh) holds d = 16 kk + 8 lh + [0, 8) of its row
    i16x8 qf[KS];
    {
      const T* qrow = static_cast<const T*>(a.q) + (int64_t)(sq.q0 + t) * a.sqn + (int64_t)(pl.kvh * G + g) * a.sqh;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
        qf[kk] = *reinterpret_cast<const i16x8*>(qrow + 16 * kk + 8 * lh) ^ (short)(a.neg_q ? 0x8000 : 0);
    }

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m_run = -INFINITY, m_lim = -INFINITY, l_run = 0.f;
    const float thr = kRescaleLog2 / sl2;

    const T* hbase = static_cast<const T*>(a.cache) + pl.kvh * a.ch;
    const int kl = sq.kv_len, P = sq.prefix;
    const int mask_cols = a.mask != nullptr ? min(min(sq.q_len, a.mask_n), kl - P) : 0;
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
        table[i] = min(max(a.seqs.kv_indices[sq.list + first_page + i], 0), a.seqs.n_pages - 1);
      if (a.mask != nullptr) {
        for (int i = tid; i < (c1 * S - ut0) * M; i += C::kWaves * 64) {
          const int row = min(pl.tile * M + i % M, TG - 1);
          words[i] = word_of((ut0 + i / M) * 32, row / G);
        }
      }
      barrier();

      // Unit j of the chunk's stream into stage j % NST.  Load i of the wave
      // moves RPL key rows (never more than a page); rows past the last key
      // repeat a valid one, so that no stale value of the pool enters P V.
      const int n = c1 - c0;
      auto issue = [&](int j) {
        const int k0 = ((c0 + j) * S + st) * 32;
        const uint32_t dst = ring + (uint32_t)((j % NST) * C::kUnit);
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
          const int u = rg * LPW + i;          // load of the unit: K's, then V's
          const bool is_v = u >= HALF;
          const int kb = (is_v ? u - HALF : u) * RPL;
          const int blk = paged::load_block(k0 + kb, RPL, kl);
          const int id = __builtin_amdgcn_readfirstlane(table[min((blk >> ps) - first_page, kTableIds - 1)]);
          const T* base = hbase + id * a.cp + (is_v ? a.cs : 0) + (int64_t)(blk & ((1 << ps) - 1)) * a.cr;
          const int row = kb + lane / CPR;
          const int from = min(lane / CPR, kl - 1 - blk);
          const int chunk = (lane % CPR) ^ (is_v ? swz_v<D>(row) : swz_k<D>(row));
          dma_1k(base, (uint32_t)from * (uint32_t)a.cr * 2u + (uint32_t)chunk * 16u, dst + (uint32_t)u * 1024u);
        }
      };

      vm_wait<0>();  // the ring's waits count its own loads alone
      for (int j = 0; j < NST - 1 && j < n; ++j) issue(j);
      for (int j = 0; j < n; ++j) {
        wait_units<LPW, NST - 2>(min(n - 1 - j, NST - 2));
        barrier();  // unit j is there, and every wave is done with unit j - 1
        if (j + NST - 1 < n) issue(j + NST - 1);

        const unsigned char* kt = smem + (st * NST + j % NST) * C::kUnit;
        const unsigned char* vt = kt + C::kTile;
        const int u = (c0 + j) * S + st;

        // S^T: lane (ln, lh) element i is key 8 (i / 4) + 4 lh + i % 4 of row ln
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          const i16x8 kf = *reinterpret_cast<const i16x8*>(kt + ln * C::kRowBytes + (((2 * kk + lh) ^ swz_k<D>(ln)) << 4));
          s = Mma<T>::run(bit_cast<V8>(kf), bit_cast<V8>(qf[kk]), s);
        }
        const bool masked = (u + 1) * 32 > P;
        uint32_t w = 0xffffffffu;
        if (masked) {
          w = a.mask != nullptr ? words[(u - ut0) * M + rg * 32 + ln] : word_of(u * 32, t);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((w >> (8 * (i >> 2) + 4 * lh + (i & 3))) & 1u)) s[i] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        const float rmax = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        // the reference point moves only when a score passes it by more than
        // 2^8 (exact for any consistent point; p stays below 2^8)
        const bool need = rmax > m_lim;
        const float m_new = need ? rmax : m_run;
        const float alpha = need ? __builtin_amdgcn_exp2f((m_run - m_new) * sl2) : 1.f;
        m_run = m_new;
        m_lim = m_new + thr;
        const float ms = m_new == -INFINITY ? 0.f : m_new;
        // P is rounded to the input type for the product with V; its row sum
        // takes the unrounded values
        float psum = 0.f;
        uint32_t pk[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f((s[i] - ms) * sl2), p1 = __builtin_amdgcn_exp2f((s[i + 1] - ms) * sl2);
          psum += p0 + p1;
          pk[i >> 1] = bit_cast<uint32_t>(T2{(T)p0, (T)p1});
        }
        l_run = l_run * alpha + psum;
        if (__ballot(need) != 0) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }

        // O^T += V^T P^T; V^T by the transposing LDS read: lane i of 16-lane
        // group x gets keys 16 s2 + 8 jj + 4 (x >> 1) + [0, 4) of
        // d = 32 dt + 16 (x & 1) + i, the key order in which P lies
        const V8 pb[2] = {bit_cast<V8>(U4{pk[0], pk[1], pk[2], pk[3]}), bit_cast<V8>(U4{pk[4], pk[5], pk[6], pk[7]})};
        const int vx = lane >> 4, vi = lane & 15;
        const int vrow = 4 * (vx >> 1) + (vi >> 2);
        const int vch = 2 * (vx & 1) + ((vi & 3) >> 1), vhalf = 8 * (vi & 1);
        const uint32_t vb = lds_addr(vt) + (uint32_t)(vrow * C::kRowBytes + vhalf);
        bool odd = false;
        if (masked) {
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
#pragma unroll
        for (int x = 0; x < 2 * DT; ++x) {
          const int dt = x >> 1, s2 = x & 1;
          i16x4 h[2];
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const int row = 16 * s2 + 8 * jj;  // swz_v has period 8 in the key
            h[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (TSFA_LDS i16x4*)(uintptr_t)(vb + (uint32_t)(row * C::kRowBytes + (((4 * dt + vch) ^ swz_v<D>(vrow)) << 4))));
          }
          i16x8 vf = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
          if (odd) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if ((vf[e] & (short)(EXP2 & 0xffff)) == (short)(EXP2 & 0xffff)) vf[e] = 0;
          }
          o[dt] = Mma<T>::run(bit_cast<V8>(vf), pb[s2], o[dt]);
        }
        if (odd) {
          for (int key = 0; key < 32; ++key) {
            if (!((w >> key) & 1u)) continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int d = 32 * dt + 8 * (i >> 2) + 4 * lh + (i & 3);
                const float v = (float)*reinterpret_cast<const T*>(vt + key * C::kRowBytes +
                                                                   (((d >> 3) ^ swz_v<D>(key)) << 4) + 2 * (d & 7));
                if (!(v - v == 0.f)) o[dt][i] += v;
              }
          }
        }
      }
      barrier();  // the rings, the table and the words are free again
      c0 = c1;
    }
    l_run += __shfl_xor(l_run, 32);

    // The streams' results join in LDS: streams 1 .. S - 1 leave (m, l, O) in
    // the ring, stream 0 takes them in.
    if constexpr (S > 1) {
      float4* jo = reinterpret_cast<float4*>(smem);                                  // [S - 1][RG][D / 8][64]
      float2* jml = reinterpret_cast<float2*>(smem + (S - 1) * RG * (D / 8) * 1024);  // [S - 1][RG][32]
      static_assert((S - 1) * RG * (D / 8) * 1024 + (S - 1) * RG * 32 * 8 <= C::kRing, "join");
      if (st > 0) {
        const int x = (st - 1) * RG + rg;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            jo[(x * (D / 8) + 4 * dt + i) * 64 + lane] =
                make_float4(o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]);
        if (lh == 0) jml[x * 32 + ln] = make_float2(m_run, l_run);
      }
      barrier();
      if (st == 0) {
#pragma unroll
        for (int s = 1; s < S; ++s) {
          const int x = (s - 1) * RG + rg;
          const float2 ml = jml[x * 32 + ln];
          const float m_new = fmaxf(m_run, ml.x);
          const float m0 = m_new == -INFINITY ? 0.f : m_new;
          const float fa = __builtin_amdgcn_exp2f((m_run - m0) * sl2), fb = __builtin_amdgcn_exp2f((ml.x - m0) * sl2);
          m_run = m_new;
          l_run = l_run * fa + ml.y * fb;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 v = jo[(x * (D / 8) + 4 * dt + i) * 64 + lane];
              o[dt][4 * i] = o[dt][4 * i] * fa + v.x * fb;
              o[dt][4 * i + 1] = o[dt][4 * i + 1] * fa + v.y * fb;
              o[dt][4 * i + 2] = o[dt][4 * i + 2] * fa + v.z * fb;
              o[dt][4 * i + 3] = o[dt][4 * i + 3] * fa + v.w * fb;
            }
        }
      }
    }

    if (st == 0) {
      if (s0 == 0 && s1 == n_steps) {
        if (r < TG) {
          const float inv = l_run > 0.f ? 1.f / l_run : (l_run == 0.f ? 0.f : l_run);  // NaN stays
          T* orow = static_cast<T*>(a.out) + (int64_t)(sq.q0 + t) * a.son + (int64_t)(pl.kvh * G + g) * a.soh;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              T4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = (T)(o[dt][4 * i + e] * inv);
              *reinterpret_cast<T4*>(orow + 32 * dt + 8 * i + 4 * lh) = v;
            }
          if (a.lse != nullptr && lh == 0)
            a.lse[(int64_t)(sq.q0 + t) * a.num_heads + pl.kvh * G + g] =
                l_run == 0.f ? -INFINITY : m_run * (sl2 * 0.6931471805599453f) + logf(l_run);
        }
      } else {
        // shared tile: slot 2 run if it began before this run, else 2 run + 1
        const int64_t slot = 2 * (int64_t)run + (s0 == 0 ? 1 : 0);
        float4* wo = a.ws_o + ((slot * RG + rg) * (D / 8)) * 64 + lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            wo[(4 * dt + i) * 64] = make_float4(o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]);
        if (lh == 0) a.ws_ml[slot * M + rg * 32 + ln] = make_float2(m_run, l_run);
        if (s0 == 0 && wave == 0 && lane == 0) {
          const int64_t last = (at + n_steps - 1) / line.per;
          a.ws_desc[run] = make_int4(b, pl.kvh, pl.tile, (int)(last - run) + 1);
        }
      }
    }

    // on along the line
    at += s1 - s0;
    if (at >= end) return;
    if constexpr (S > 1) barrier();  // the ring is written again
    pl.step = 0;
    if (++pl.tile == paged::cut_tiles(cut, sq)) {
      pl.tile = 0;
      if (++pl.kvh == cut.num_kv_heads) {
        pl.kvh = 0;
        do {
          if (++pl.b >= a.seqs.batch) return;  // not reached: steps are left, so some sequence has them
          pl.seq = paged::seq_of(a.seqs, pl.b);
        } while (paged::cut_tiles(cut, pl.seq) == 0);
      }
    }
  }
}

// Joins the parts of the tiles that several runs share: block (run, row
// group); wave w takes d tiles w, w + 4, ...
template <typename T, int D, int RG>
__global__ __launch_bounds__(256) void combine_kernel(const Args a) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int run = blockIdx.x, rg = blockIdx.y;
  const int4 desc = a.ws_desc[run];
  const int parts = desc.w;
  if (parts == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 31, lh = lane >> 5;
  constexpr int M = 32 * RG;
  const Seq sq = paged::seq_of(a.seqs, desc.x);
  const int G = a.cut.group, TG = sq.q_len * G;
  const int r = desc.z * M + rg * 32 + ln;
  if (r >= TG) return;
  const int t = r / G, g = r - t * G;
  auto slot_of = [&](int p) { return p == 0 ? 2 * (int64_t)run + 1 : 2 * (int64_t)(run + p); };
  const float2* ml = a.ws_ml + rg * 32 + ln;
  float m = -INFINITY;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, ml[slot_of(p) * M].x);
  const float m0 = m == -INFINITY ? 0.f : m, sl2 = a.scale_log2;
  for (int dt = wave; dt < D / 32; dt += 4) {
    float l = 0.f;
    float4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < parts; ++p) {
      const int64_t slot = slot_of(p);
      const float2 x = ml[slot * M];
      const float f = __builtin_amdgcn_exp2f((x.x - m0) * sl2);
      l += x.y * f;
      const float4* wo = a.ws_o + ((slot * RG + rg) * (D / 8) + 4 * dt) * 64 + lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = wo[i * 64];
        o[i].x += v.x * f;
        o[i].y += v.y * f;
        o[i].z += v.z * f;
        o[i].w += v.w * f;
      }
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int h = desc.y * G + g;
    T* orow = static_cast<T*>(a.out) + (int64_t)(sq.q0 + t) * a.son + (int64_t)h * a.soh + 32 * dt + 4 * lh;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T4 v = {(T)(o[i].x * inv), (T)(o[i].y * inv), (T)(o[i].z * inv), (T)(o[i].w * inv)};
      *reinterpret_cast<T4*>(orow + 8 * i) = v;
    }
    if (a.lse != nullptr && dt == 0 && lh == 0)
      a.lse[(int64_t)(sq.q0 + t) * a.num_heads + h] = l == 0.f ? -INFINITY : m * (sl2 * 0.6931471805599453f) + logf(l);
  }
}

struct Sizes {
  int groups, few_rows;
  size_t o, ml, desc;
  size_t total() const { return o + ml + desc; }
};

// 32-row tiles with four key streams where a sequence has at most 32 rows on
// average, else 128-row tiles with two.
inline Sizes sizes_of(int cus, int batch, int total_q, int num_heads, int num_kv_heads, int head_dim) {
  Sizes s;
  const int64_t rows = (int64_t)total_q * (num_heads / num_kv_heads);
  s.few_rows = rows <= (int64_t)32 * batch;
  s.groups = cus;
  const int m = s.few_rows ? 32 : 128;
  s.o = align256((size_t)2 * s.groups * m * head_dim * 4);
  s.ml = align256((size_t)2 * s.groups * m * 8);
  s.desc = align256((size_t)s.groups * 16);
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
  hipLaunchKernelGGL((combine_kernel<T, D, RG>), dim3((unsigned)a.groups, RG), dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? TSFA_OK : TSFA_ERR_LAUNCH;
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
  return varlen::sizes_of(cus, batch, total_q, num_heads, num_kv_heads, head_dim).total();
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
  // a lane's row offset within a page is an unsigned 32-bit byte count
  if (cache_strides[4] != 1 || cache_strides[2] < 0 || cache_strides[2] > ((int64_t)1 << 26)) return TSFA_ERR_UNSUPPORTED;
  if (batch == 0 || total_q == 0) return TSFA_OK;
  for (const void* p : {q, kv_cache, (const void*)o}) {
    if (p == nullptr) return TSFA_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return TSFA_ERR_UNSUPPORTED;
  }
  if (q_indptr == nullptr || kv_lens == nullptr || kv_indices == nullptr) return TSFA_ERR_INVALID_ARGUMENT;
  int cus = 0;
  if (device_cu_count(&cus) != TSFA_OK) return TSFA_ERR_DEVICE;
  const varlen::Sizes sz = varlen::sizes_of(cus, batch, total_q, num_heads, num_kv_heads, head_dim);
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
  a.cut.rows = sz.few_rows ? 32 : 128;
  a.cut.keys = sz.few_rows ? 128 : 64;
  a.cut.group = num_heads / num_kv_heads;
  a.cut.num_kv_heads = num_kv_heads;
  a.cut.causal = mask == nullptr;
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
  a.ws_desc = reinterpret_cast<int4*>(ws + sz.o + sz.ml);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TSFA_DTYPE_BF16) {
    if (head_dim == 128) return sz.few_rows ? varlen::launch<__bf16, 128, 4, 1>(a, s) : varlen::launch<__bf16, 128, 2, 4>(a, s);
    return sz.few_rows ? varlen::launch<__bf16, 64, 4, 1>(a, s) : varlen::launch<__bf16, 64, 2, 4>(a, s);
  }
  if (head_dim == 128) return sz.few_rows ? varlen::launch<_Float16, 128, 4, 1>(a, s) : varlen::launch<_Float16, 128, 2, 4>(a, s);
  return sz.few_rows ? varlen::launch<_Float16, 64, 4, 1>(a, s) : varlen::launch<_Float16, 64, 2, 4>(a, s);
}
