// Drafted tokens enter the paged K/V pool: queries and keys rotated by their
// positions, keys and values written to their pages, in one pass.
//
// For token n of sequence b and pair i of the rotated part of a head,
//   a = positions[n] * inv_freq[i],  (x1, x2) -> s (x1 cos a - x2 sin a, x2 cos a + x1 sin a)
// with s the attention scaling; pair i is (i, rot/2 + i) or, interleaved,
// (2i, 2i + 1).  The angle is formed in 64 bits and reduced to a turn there:
// a 32-bit product is off by 0.06 rad a million tokens out.
//
// Bound by memory: every element is read once and written once, 16 bytes a
// lane, a workgroup to a token whose waves deal the heads' 16-element slots
// among them; a lane holds both elements of its pairs, so q may be rotated in
// place.  7800 tokens of 64 + 2 * 8 heads of 128 (332 MB): 66 us, 5.0 TB/s, what
// a copy of that size reaches; 700 tokens of 32 + 2 * 8 heads 6.5 us; one token
// 3.7 us, of which about 2 are an empty launch.
#include <hip/hip_runtime.h>

#include "tsfa_internal.h"
#include "tsfa_paged.h"

namespace tsfa {
namespace append {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;  // pairs of a head

struct Args {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  void* cache;
  const void* positions;
  const float* inv_freq;
  paged::Seqs seqs;
  int64_t sqn, sqh, skn, skh, svn, svh, son, soh;  // elements
  int64_t cp, cs, cr, ch;                          // cache: page, K/V slot, row, head
  float scale;
  int num_heads, num_kv_heads, head_dim, half;
  int pos64, interleaved;
};

template <typename T> __device__ inline float to_f(T x) { return (float)x; }

// The sequence of token n: the last b with q_indptr[b] <= n.
__device__ inline int seq_at(const paged::Seqs& s, int n) {
  int lo = 0, hi = s.batch;  // q_indptr[lo] <= n < q_indptr[hi] in a valid call
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.q_indptr[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void append_kernel(const Args a) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  __shared__ float2 turn[kThreads / 64][kMaxHalf];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x;
  const int b = seq_at(a.seqs, n);
  const paged::Seq s = paged::seq_of(a.seqs, b);
  if (n < s.q0 || n >= s.q0 + s.q_len) return;  // behind the last sequence

  const double pos = a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[n]
                             : (double)static_cast<const int32_t*>(a.positions)[n];
  for (int i = lane; i < a.half; i += 64) {
    const double turns = pos * (double)a.inv_freq[i] * 0.15915494309189535;  // 1 / (2 pi)
    float sn, cs;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    turn[wave][i] = make_float2(cs * a.scale, sn * a.scale);
  }
  // the wave's lanes read each other's entries (every wave forms the token's
  // angles: no barrier)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

  // the key's place in the pool; tokens without one are not written
  const int64_t kv_len = a.seqs.kv_lens[b];
  const int64_t key = kv_len - s.q_len + (n - s.q0);
  T* krow = nullptr;
  if (key >= 0 && (key >> a.seqs.page_shift) < s.pages) {
    const int page = a.seqs.kv_indices[s.list + (key >> a.seqs.page_shift)];
    if (page >= 0 && page < a.seqs.n_pages)
      krow = static_cast<T*>(a.cache) + page * a.cp + (key & ((1 << a.seqs.page_shift) - 1)) * a.cr;
  }

  const int sph = a.head_dim / 16, rots = a.half / 8;  // 16-element slots of a head, rotated ones
  const int hk = a.num_heads + a.num_kv_heads, total = (hk + a.num_kv_heads) * sph;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int h = i / sph, c = i - h * sph;
    const bool rotate = h < hk && c < rots;
    const bool halves = rotate && !a.interleaved;
    const int da = halves ? 8 * c : 16 * c, db = halves ? a.half + 8 * c : 16 * c + 8;
    const T* src;
    T* dst;
    if (h < a.num_heads) {
      src = static_cast<const T*>(a.q) + n * a.sqn + h * a.sqh;
      dst = static_cast<T*>(a.out) + n * a.son + h * a.soh;
    } else {
      const int kh = h < hk ? h - a.num_heads : h - hk;
      src = h < hk ? static_cast<const T*>(a.k) + n * a.skn + kh * a.skh
                   : static_cast<const T*>(a.v) + n * a.svn + kh * a.svh;
      if (krow == nullptr) continue;
      dst = krow + kh * a.ch + (h < hk ? 0 : a.cs);
    }
    T8 xa = *reinterpret_cast<const T8*>(src + da), xb = *reinterpret_cast<const T8*>(src + db);
    if (rotate) {
      const float2* tr = &turn[wave][8 * c];
      if (halves) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x1 = to_f(xa[e]), x2 = to_f(xb[e]);
          xa[e] = (T)(x1 * tr[e].x - x2 * tr[e].y);
          xb[e] = (T)(x2 * tr[e].x + x1 * tr[e].y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 ta = tr[e / 2], tb = tr[4 + e / 2];
          const float a1 = to_f(xa[e]), a2 = to_f(xa[e + 1]), b1 = to_f(xb[e]), b2 = to_f(xb[e + 1]);
          xa[e] = (T)(a1 * ta.x - a2 * ta.y);
          xa[e + 1] = (T)(a2 * ta.x + a1 * ta.y);
          xb[e] = (T)(b1 * tb.x - b2 * tb.y);
          xb[e + 1] = (T)(b2 * tb.x + b1 * tb.y);
        }
      }
    }
    *reinterpret_cast<T8*>(dst + da) = xa;
    *reinterpret_cast<T8*>(dst + db) = xb;
  }
}

}  // namespace append
}  // namespace tsfa

using namespace tsfa;

extern "C" int tsfa_append_paged_kv(const void* q, const void* k, const void* v, void* out, void* kv_cache,
                                    const void* positions, int positions_64, const float* inv_freq, int rot_dim,
                                    int interleaved, float attention_scaling, const int32_t* q_indptr,
                                    const int32_t* kv_lens, const int32_t* kv_indptr, const int32_t* kv_indices,
                                    int64_t n_indices, int64_t page_table_stride, int page_table_width, int n_pages,
                                    int page_size, const int64_t* strides, const int64_t* cache_strides, int batch,
                                    int total_q, int num_heads, int num_kv_heads, int head_dim, int dtype,
                                    tsfa_stream_t stream) {
  if (batch < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || strides == nullptr || cache_strides == nullptr)
    return TSFA_ERR_INVALID_ARGUMENT;
  if (rot_dim < 0 || rot_dim > head_dim) return TSFA_ERR_INVALID_ARGUMENT;
  if (dtype != TSFA_DTYPE_FP16 && dtype != TSFA_DTYPE_BF16) return TSFA_ERR_UNSUPPORTED;
  if (head_dim <= 0 || head_dim % 16 != 0 || head_dim > 256 || rot_dim % 16 != 0) return TSFA_ERR_UNSUPPORTED;
  if (num_heads > 65536 || num_kv_heads > 65536 || total_q > 1 << 23) return TSFA_ERR_UNSUPPORTED;
  const int st = paged_check(kv_indptr, n_indices, page_table_stride, page_table_width, n_pages, page_size, batch);
  if (st != TSFA_OK) return st;
  // rows the kernel reads and writes 16 bytes at a time
  for (int i = 0; i < 4; ++i)
    if (strides[3 * i + 2] != 1 || strides[3 * i] % 8 != 0 || strides[3 * i + 1] % 8 != 0) return TSFA_ERR_UNSUPPORTED;
  if (cache_strides[4] != 1) return TSFA_ERR_UNSUPPORTED;
  for (int i = 0; i < 4; ++i)
    if (cache_strides[i] % 8 != 0) return TSFA_ERR_UNSUPPORTED;
  if (batch == 0 || total_q == 0) return TSFA_OK;
  const void* ptrs[5] = {q, k, v, out, kv_cache};
  for (const void* p : ptrs) {
    if (p == nullptr) return TSFA_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return TSFA_ERR_UNSUPPORTED;
  }
  if (positions == nullptr || q_indptr == nullptr || kv_lens == nullptr || (kv_indices == nullptr && n_indices > 0) ||
      (rot_dim > 0 && inv_freq == nullptr))
    return TSFA_ERR_INVALID_ARGUMENT;

  append::Args a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.cache = kv_cache;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.seqs = make_seqs(q_indptr, kv_lens, kv_indptr, kv_indices, n_indices, page_table_stride, page_table_width, n_pages,
                     page_size, batch, total_q);
  a.sqn = strides[0], a.sqh = strides[1];
  a.skn = strides[3], a.skh = strides[4];
  a.svn = strides[6], a.svh = strides[7];
  a.son = strides[9], a.soh = strides[10];
  a.cp = cache_strides[0], a.cs = cache_strides[1], a.cr = cache_strides[2], a.ch = cache_strides[3];
  a.scale = attention_scaling;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.half = rot_dim / 2;
  a.pos64 = positions_64 != 0;
  a.interleaved = interleaved != 0;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TSFA_DTYPE_BF16)
    hipLaunchKernelGGL((append::append_kernel<__bf16>), dim3((unsigned)total_q), dim3(append::kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((append::append_kernel<_Float16>), dim3((unsigned)total_q), dim3(append::kThreads), 0, s, a);
  return hipGetLastError() == hipSuccess ? TSFA_OK : TSFA_ERR_LAUNCH;
}
