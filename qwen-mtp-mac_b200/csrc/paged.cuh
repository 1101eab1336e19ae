// Shared pieces of the paged-cache kernels (paged.cu, paged_prompt.cu): the device view of a cache,
// which keys a query sees, and the strict evaluation of one attention row.
#pragma once
#include <atomic>
#include <cmath>

#include "common.cuh"

namespace qmtp {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxSeqs = 4096;
constexpr int kMaxHeads = 65536;

// Device view of qmtp_paged_cache.  page = 1 << page_log.
struct PagedView {
  uint16_t* k;
  uint16_t* v;
  const int* table;
  const int* lens;
  long long pages, ld_table;
  int nkv, page_log, table_w, B;
};

// Which keys a query at position p sees (qmtp_paged_args): j <= p and (no window, or p - j < window, or j < sinks).
struct Visible {
  int window, sinks;
  __device__ __forceinline__ bool operator()(int p, int j) const {
    return j <= p && (window == 0 || p - j < window || j < sinks);
  }
  // first key of the window of the query at position p (0 without a window)
  __device__ __forceinline__ int first(int p) const { return window == 0 || window > p ? 0 : p - window + 1; }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Two fp32 values in a 64-bit register and the packed arithmetic on them.
__device__ __forceinline__ uint64_t f2_pack(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Length of sequence b: a value the table cannot hold counts as empty (and is reported).
__device__ __forceinline__ int seq_len(const PagedView& c, int b, unsigned* err) {
  const int n = c.lens[b];
  if (n < 0 || n > ((long long)c.table_w << c.page_log)) {
    if (err) atomicOr(err, DEVERR_BADARG);
    return 0;
  }
  return n;
}

// Row index (of Dh elements) of position j of sequence b, head kh, in k and v; -1 for a bad page.
__device__ __forceinline__ long long cache_row(const PagedView& c, int b, int kh, int j, unsigned* err) {
  const long long pg = c.table[(long long)b * c.ld_table + (j >> c.page_log)];
  if (pg < 0 || pg >= c.pages) {
    atomicOr(err, DEVERR_BADARG);
    return -1;
  }
  return ((pg * c.nkv + kh) << c.page_log) + (j & ((1 << c.page_log) - 1));
}

// N consecutive bf16 values (N 2, 4 or 8, aligned to their size), two a word.
template <int N>
__device__ __forceinline__ void load_dims(uint32_t (&w)[N / 2], const uint16_t* p) {
  if constexpr (N == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// One query row over the keys [j0, j1) of its sequence that it sees, by one warp: lane l owns dims
// [l * Dh / 32, (l + 1) * Dh / 32).  One pass with the running maximum m (base 2), sum l and numerator o of
// the softmax, which the caller starts at (-inf, 0, 0).  Only rows that are seen are read, so nothing
// behind the mask can reach o.  The rows of eight keys are on their way at once.
template <int Dh>
__device__ __noinline__ void attend_row_strict(const PagedView c, const uint16_t* __restrict__ qrow, int b, int kh,
                                               int p, int j0, int j1, Visible vis, float scale2, unsigned* err,
                                               float& m, float& l, float (&o)[Dh / 32]) {
  constexpr int N = Dh / 32, AHEAD = 8;
  const int lane = threadIdx.x & 31, end = min(j1, p + 1);
  float q[N];
#pragma unroll
  for (int e = 0; e < N; ++e) q[e] = bf2f(qrow[lane * N + e]);
  for (int j = j0; j < end; j += AHEAD) {
    const bool sees = lane < AHEAD && j + lane < end && vis(p, j + lane);
    const unsigned seen = __ballot_sync(0xFFFFFFFFu, sees);
    if (seen == 0) continue;
    const long long row = sees ? cache_row(c, b, kh, j + lane, err) : -1;
    uint32_t k[AHEAD][N / 2], v[AHEAD][N / 2];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const long long r = __shfl_sync(0xFFFFFFFFu, row, i);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) k[i][e] = v[i][e] = 0;
      if (r >= 0) {
        load_dims<N>(k[i], c.k + r * Dh + lane * N);
        load_dims<N>(v[i], c.v + r * Dh + lane * N);
      }
    }
    float s[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) s[i] = __fmaf_rn(q[e], e & 1 ? bfhi(k[i][e / 2]) : bflo(k[i][e / 2]), s[i]);
      s[i] = __fmul_rn(warp_sum(s[i]), scale2);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (!(seen >> i & 1)) continue;
      const float mn = fmaxf(m, s[i]);
      const float safe = mn == -INFINITY ? 0.0f : mn;
      const float a = exp2f(__fsub_rn(m, safe)), w = exp2f(__fsub_rn(s[i], safe));
      l = __fmaf_rn(l, a, w);
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = __fmaf_rn(w, e & 1 ? bfhi(v[i][e / 2]) : bflo(v[i][e / 2]), __fmul_rn(o[e], a));
      m = mn;
    }
  }
}

// What a CTA's barrier waits share, in shared memory.  A wait gives up after 2^20 polls without a sign of life from a warp
// that is at long work of its own (rows computed by the definition); the others then give up soon too.
struct WaitState {
  int dead;   // a wait has run out (the error word tells)
  int alive;  // counts the signs
};
__device__ __forceinline__ bool given_up(const WaitState* w) { return *reinterpret_cast<const volatile int*>(&w->dead) != 0; }
__device__ __forceinline__ void sign_of_life(WaitState* w) {
  if ((threadIdx.x & 31) == 0) atomicAdd(&w->alive, 1);
}

// A bounded barrier wait.  False: gave up.
__device__ __forceinline__ bool bar_wait_slow(WaitState* w, uint64_t* bar, uint32_t parity, unsigned* err) {
  const volatile int* alive = &w->alive;
  int last = *alive;
#pragma unroll 1
  for (uint32_t it = 0; it < (1u << 20); ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63) == 63) {
      if (given_up(w)) return false;
      const int now = *alive;
      if (now != last) it = 0;
      last = now;
    }
  }
  atomicOr(err, DEVERR_TIMEOUT);
  *reinterpret_cast<volatile int*>(&w->dead) = 1;
  return false;
}
__device__ __forceinline__ bool bar_wait(WaitState* w, uint64_t* bar, uint32_t parity, unsigned* err) {
  return mbar_try_wait(bar, parity) || bar_wait_slow(w, bar, parity, err);
}
// By every lane of a warp, which is converged afterwards.
__device__ __forceinline__ bool warp_wait(WaitState* w, uint64_t* bar, uint32_t parity, unsigned* err) {
  return __all_sync(0xFFFFFFFFu, bar_wait(w, bar, parity, err));
}

__device__ __forceinline__ void prefetch_tensormap(const void* tmap) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(tmap) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Runs a set-up call (a kernel's attributes) once for every device the process uses; false if it failed,
// and a failure is tried again by the next call.
struct DeviceOnce {
  std::atomic<bool> done[64] = {};
  template <typename F>
  bool operator()(F f) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done[dev].load(std::memory_order_acquire)) return true;
    if (f() != cudaSuccess) return false;
    done[dev].store(true, std::memory_order_release);
    return true;
  }
};

// bf16 tensor map with 128-byte swizzle (boxes 64 elements wide); what lies outside reads as zeros.
inline bool encode_pages(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Host checks shared by the entry points; fills the device view.
int paged_view(const qmtp_paged_cache* cache, PagedView* out);
int paged_check_args(const qmtp_paged_args* a, const qmtp_paged_cache* c);

}  // namespace qmtp
