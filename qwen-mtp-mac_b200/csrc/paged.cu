// Paged key/value cache: the writer (per-head q/k norm + rotation + append) and the attention of the
// newest tokens, split over the cache's length and joined.  The prompt form is in paged_prompt.cu.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace qmtp {

// ----------------------------------------------------------------------------- append
// Per head row x of q or k: y = x / sqrt(mean x^2 + eps) * w, then dims (i, i + R/2), i < R/2, turn by the
// position's angle: (y_i c - y_j s, y_j c + y_i s).  All fp32; one rounding to bf16 on the way out.
// A group of Dh / 8 lanes owns a row (16 bytes a lane); a warp takes 4 steps of 32 / (Dh / 8) head rows of
// one token, loads all of them first and shares the token's angles.  Bound: HBM (one read, one write).
struct AppendArgs {
  const uint16_t* qkv;
  long long ld;
  const int* cu;
  const uint16_t *qw, *kw;
  const float *cos_t, *sin_t;
  uint16_t* q_out;
  float eps;
  int T, S, nq, gated, rotary, max_pos;
  unsigned* err;
};

constexpr int kAppendSteps = 4;

template <int Dh>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedView c, AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int LPR = Dh / 8, RPS = 32 / LPR;  // lanes per row, rows per step
  const int lane = threadIdx.x & 31, sub = lane % LPR;
  const int heads = a.nq + 2 * c.nkv;
  const int units = (heads + kAppendSteps * RPS - 1) / (kAppendSteps * RPS);  // warps per token
  const long long wid = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = int(wid / units);
  const int h0 = int(wid - (long long)t * units) * kAppendSteps * RPS + lane / LPR;
  if (t >= a.T) return;
  const uint16_t* row = a.qkv + (long long)t * a.ld;
  uint4 x[kAppendSteps];
#pragma unroll
  for (int i = 0; i < kAppendSteps; ++i) {
    const int h = h0 + i * RPS;
    if (h < heads) {
      const long long head = h < a.nq ? (a.gated ? 2 * h : h) : (a.gated ? a.nq + h : h);
      x[i] = *reinterpret_cast<const uint4*>(row + head * Dh + 8 * sub);
    }
  }
  // the row's sequence and position
  int b, p;
  if (a.cu == nullptr) {
    b = t / a.S;
    p = seq_len(c, b, a.err) - a.S + (t - b * a.S);
  } else {
    // sequences that end at or before row t, counted a warp at a time (cu does not decrease)
    b = 0;
    for (int i = 0; i < c.B; i += 32) {
      const int k = i + lane;
      b += __popc(__ballot_sync(0xFFFFFFFFu, k < c.B && a.cu[k + 1] <= t));
    }
    if (b >= c.B || t < a.cu[b]) return;  // a row of no sequence
    p = seq_len(c, b, a.err) - a.cu[b + 1] + t;
  }
  if (p < 0) return;
  const bool far = a.cos_t != nullptr && p >= a.max_pos;
  if (far || (p >> c.page_log) >= c.table_w) {
    if (lane == 0) atomicOr(a.err, DEVERR_BADARG);
    return;
  }
  const int half = a.rotary / 2;
  float cs[8], sn[8];
  const int d0 = 8 * sub, i0 = d0 < half ? d0 : d0 - half;
  const bool turns = a.cos_t != nullptr && d0 < a.rotary;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    float4 cv = make_float4(1.f, 1.f, 1.f, 1.f), sv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turns) {
      cv = *reinterpret_cast<const float4*>(a.cos_t + (long long)p * half + i0 + e);
      sv = *reinterpret_cast<const float4*>(a.sin_t + (long long)p * half + i0 + e);
    }
    cs[e] = cv.x; cs[e + 1] = cv.y; cs[e + 2] = cv.z; cs[e + 3] = cv.w;
    sn[e] = sv.x; sn[e + 1] = sv.y; sn[e + 2] = sv.z; sn[e + 3] = sv.w;
  }
  const int lane_p = turns ? lane + (d0 < half ? half / 8 : -(half / 8)) : lane;
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (a.qw) wq = *reinterpret_cast<const uint4*>(a.qw + 8 * sub);
  if (a.kw) wk = *reinterpret_cast<const uint4*>(a.kw + 8 * sub);
#pragma unroll
  for (int i = 0; i < kAppendSteps; ++i) {
    const int h = h0 + i * RPS;
    const bool live = h < heads, isq = h < a.nq, isv = h >= a.nq + c.nkv;
    float y[8];
    const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { y[2 * e] = live ? bflo(u[e]) : 0.f; y[2 * e + 1] = live ? bfhi(u[e]) : 0.f; }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __fmaf_rn(y[e], y[e], ss);
#pragma unroll
    for (int d = LPR / 2; d >= 1; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, d));
    if ((isq ? a.qw : a.kw) != nullptr) {
      const float r = rsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.0f / Dh), a.eps));
      const uint4 w4 = isq ? wq : wk;
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(__fmul_rn(y[e], r), (e & 1) ? bfhi(w[e >> 1]) : bflo(w[e >> 1]));
    }
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl_sync(0xFFFFFFFFu, y[e], lane_p);
      o[e] = y[e];
      if (turns) o[e] = __fmaf_rn(y[e], cs[e], d0 < half ? -__fmul_rn(other, sn[e]) : __fmul_rn(other, sn[e]));
    }
    if (!live) continue;
    uint4 r4 = x[i];
    if (!isv) {
      uint32_t pk[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pk[e] = f2bf(o[2 * e]) | (uint32_t(f2bf(o[2 * e + 1])) << 16);
      r4 = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    }
    if (isq) {
      *reinterpret_cast<uint4*>(a.q_out + ((long long)t * a.nq + h) * Dh + d0) = r4;
    } else {
      const long long r = cache_row(c, b, isv ? h - a.nq - c.nkv : h - a.nq, p, a.err);
      if (r >= 0) *reinterpret_cast<uint4*>((isv ? c.v : c.k) + r * Dh + d0) = r4;
    }
  }
}

// ----------------------------------------------------------------------------- decode attention
// A unit of work is (sequence, slab of keys, key head, tile of query rows); rows are the S tokens x G query
// heads of the key head.  Scores and the weighted sum run on the tensor cores with the keys (dims) on the
// M side, S^T = K Q^T and O^T = V^T P^T (m16n8k16), so a group of 4 or 8 rows fills the 8-wide N side.
// The keys' bytes bound it (4 flops a byte and row group), so mma.sync, fed from a ring that cp.async
// keeps full, is enough: its pipe is a small part of the time the bytes take.
constexpr int kTile = 64;      // keys per step: 16 a warp for the scores
constexpr int kRing = 3;       // ring entries: a tile of K or of V each
constexpr int kFineSlab = 128; // slab sizes: see slab_of
constexpr int kFineKeys = 4096;
constexpr int kSlab = 512;
constexpr int kMaxS = 8;

// Slabs have fixed positions: [0, 4096) in slabs of 128, then slabs of 512; 128 everywhere (fine) for windows up to
// 4096.  Fine slabs spread a short context over the SMs (4 key heads x 2048 keys: 64 units); large ones keep the
// partial results (Dh + 2 floats a row and slab) small next to the keys of a long one.  Fixed positions make a
// row's arithmetic independent of the batch and of the call's other rows.
__host__ __device__ inline int slab_of(int j, bool fine) {
  return fine || j < kFineKeys ? j / kFineSlab : kFineKeys / kFineSlab + (j - kFineKeys) / kSlab;
}
__device__ __forceinline__ int slab_begin(int i, bool fine) {
  return fine || i <= kFineKeys / kFineSlab ? i * kFineSlab : kFineKeys + (i - kFineKeys / kFineSlab) * kSlab;
}

struct DecodeArgs {
  const uint16_t *q, *gate;
  uint16_t* out;
  long long q_ld, gate_ld, gate_hs;
  float* ws_o;    // [B][max_slabs][S * nq][Dh] numerators
  float2* ws_ml;  // [B][max_slabs][S * nq] running maximum (base 2) and sum
  int nq, S, G, row_tiles, max_slabs, fine;
  float scale2;   // scale * log2(e)
  Visible vis;
  unsigned* err;
};

// Slabs of one sequence that some query row of it sees: [0, first) and [from, from + count - first).
struct SlabList {
  int len, lo, first, from, count;
};
__device__ __forceinline__ SlabList slab_list(const PagedView& c, const DecodeArgs& a, int b, unsigned* err) {
  SlabList s;
  s.len = seq_len(c, b, err);
  s.lo = a.vis.first(max(0, s.len - a.S));  // the first key of the oldest row's window
  s.from = slab_of(s.lo, a.fine);
  s.first = a.vis.sinks > 0 && s.lo > 0 ? min(slab_of(min(a.vis.sinks, s.lo) - 1, a.fine) + 1, s.from) : 0;
  s.count = s.len > 0 ? s.first + slab_of(s.len - 1, a.fine) + 1 - s.from : 1;  // an empty sequence: one empty slab
  return s;
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte asynchronous copy; zeros when !live
__device__ __forceinline__ void cp_async16_z(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int Dh, int NT>
struct DecodeSmem {
  uint16_t kv[kRing][kTile * Dh];  // 16-byte chunk x of row r sits at chunk x ^ (r & 7)
  uint16_t p[8 * NT][kTile + 8];   // weights, [row][key]
  float mx[4][8 * NT];
  float sum[4][8 * NT];
  int scan[4];
  int bad;
};

template <int Dh, int NT>
__global__ void __launch_bounds__(128, Dh == 256 ? 2 : 4) paged_decode_kernel(PagedView c, DecodeArgs a) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DecodeSmem<Dh, NT>& sm = *reinterpret_cast<DecodeSmem<Dh, NT>*>(smem_raw);
  int* s_pre = reinterpret_cast<int*>(smem_raw + sizeof(DecodeSmem<Dh, NT>));  // [B + 1] slabs before sequence b
  constexpr int CPR = Dh / 8;        // 16-byte chunks per row
  constexpr int RPI = 32 / CPR;      // rows a warp copies per instruction
  constexpr int MT = Dh / 64;        // 16-dim tiles of a warp in the weighted sum
  constexpr float kNone = -INFINITY;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane & 3, oct = lane >> 2;
  // slabs before every sequence
  int total = 0;
  for (int b0 = 0; b0 < c.B; b0 += 128) {
    const int b = b0 + tid;
    const int n = b < c.B ? slab_list(c, a, b, blockIdx.x == 0 ? a.err : nullptr).count : 0;
    int chunk;
    const int before = block_excl_scan(n, sm.scan, chunk);
    if (b < c.B) s_pre[b] = total + before;
    total += chunk;
  }
  if (tid == 0) s_pre[c.B] = total;
  __syncthreads();
  const int R = a.S * a.G, per = c.nkv * a.row_tiles;
  const long long units = (long long)total * per;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int slab_g = int(u / per), rest = int(u - (long long)slab_g * per);
    const int kh = rest / a.row_tiles, row0 = (rest - kh * a.row_tiles) * 8 * NT;
    int b = 0;  // the last sequence that begins at or before this slab
    for (int step = 1 << (31 - __clz(c.B)); step > 0; step >>= 1)
      if (b + step < c.B && s_pre[b + step] <= slab_g) b += step;
    const SlabList sl = slab_list(c, a, b, nullptr);
    const int i_slab = slab_g - s_pre[b];
    const int slab = i_slab < sl.first ? i_slab : sl.from + i_slab - sl.first;
    const int k_begin = slab_begin(slab, a.fine), k_end = min(slab_begin(slab + 1, a.fine), sl.len);
    const int pos0 = sl.len - a.S;
    // tiles of the slab that hold a needed key
    auto next_tile = [&](int j) {
      while (j < k_end && a.vis.window != 0 && j + kTile <= sl.lo && j >= a.vis.sinks) j += kTile;
      return j;
    };
    // rows of this lane: n = 8 t + 2 quad + e (softmax, output), n = 8 t + oct (query fragment)
    uint32_t qf[NT][Dh / 16][2];
    int prow[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + 8 * t + 2 * quad + e;
        prow[t][e] = r < R ? pos0 + r / a.G : -1;
      }
      const int r = row0 + 8 * t + oct;
      const int s = r / a.G;
      const uint16_t* qp = a.q + (long long)(b * a.S + s) * a.q_ld + (long long)(kh * a.G + r - s * a.G) * Dh + 2 * quad;
#pragma unroll
      for (int k = 0; k < Dh / 16; ++k) {
        qf[t][k][0] = r < R ? *reinterpret_cast<const uint32_t*>(qp + 16 * k) : 0u;
        qf[t][k][1] = r < R ? *reinterpret_cast<const uint32_t*>(qp + 16 * k + 8) : 0u;
      }
    }
    // row of the caches that this lane's key (16 warp + lane % 16) of the tile at j lies in, -1: none needed
    auto key_row = [&](int j) -> long long {
      const int key = j + 16 * warp + (lane & 15);
      if (key >= k_end || (a.vis.window != 0 && key < sl.lo && key >= a.vis.sinks)) return -1;
      return cache_row(c, b, kh, key, a.err);
    };
    auto load = [&](int slot, const uint16_t* base, long long r_lane) {
      const uint32_t dst = smem_u32(sm.kv[slot]);
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const int rr = i * RPI + lane / CPR;  // row of the warp's 16
        const long long r = __shfl_sync(0xFFFFFFFFu, r_lane, rr);
        const int row = 16 * warp + rr, ch = lane % CPR;
        cp_async16_z(dst + row * Dh * 2 + ((ch ^ (row & 7)) << 4), base + (r < 0 ? 0 : r) * Dh + ch * 8, r >= 0);
      }
    };
    // ring order K0 V0 K1 V1 ...; entry e in slot e % 3.  Two entries ahead of the one in use.
    int j = next_tile(k_begin), j_next = j < k_end ? next_tile(j + kTile) : j;
    long long r_cur = j < k_end ? key_row(j) : -1, r_next = j_next < k_end ? key_row(j_next) : -1;
    int slot = 0;  // slot of K of the current tile
    if (j < k_end) {
      load(0, c.k, r_cur);
      cp_async_commit();
      load(1, c.v, r_cur);
    }
    cp_async_commit();
    float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = kNone;
      l[t][0] = l[t][1] = 0.0f;
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][t][e] = 0.0f;
    }
    while (j < k_end) {
      const int sv = slot + 1 == kRing ? 0 : slot + 1, sk2 = sv + 1 == kRing ? 0 : sv + 1;
      cp_async_wait<1>();
      __syncthreads();  // K has landed; the previous tile's V is free
      if (j_next < k_end) load(sk2, c.k, r_next);
      cp_async_commit();
      // scores of this warp's 16 keys
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.0f;
      {
        const int row = 16 * warp + (lane & 15);
        const uint32_t base = smem_u32(sm.kv[slot]) + row * Dh * 2;
#pragma unroll
        for (int k = 0; k < Dh / 16; ++k) {
          uint32_t af[4];
          ldsm_x4(af, base + (((2 * k + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_bf16(s[t], af, qf[t][k][0], qf[t][k][1]);
        }
      }
      const bool all = j + kTile - 1 <= pos0 && (a.vis.window == 0 || j >= a.vis.first(sl.len - 1));
      float mn[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = j + 16 * warp + oct + 8 * (e >> 1);
          s[t][e] = all || a.vis(prow[t][e & 1], key) ? __fmul_rn(s[t][e], a.scale2) : kNone;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[t][e], s[t][e + 2]);
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
          if (oct == 0) sm.mx[warp][8 * t + 2 * quad + e] = x;
        }
      }
      __syncthreads();  // K is free
      float alpha[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = 8 * t + 2 * quad + e;
          mn[t][e] = fmaxf(fmaxf(m[t][e], fmaxf(sm.mx[0][n], sm.mx[1][n])), fmaxf(sm.mx[2][n], sm.mx[3][n]));
          const float safe = mn[t][e] == kNone ? 0.0f : mn[t][e];  // nothing seen yet: every weight is 0
          alpha[t][e] = ex2(__fsub_rn(m[t][e], safe));
          m[t][e] = mn[t][e];
          const float p0 = ex2(__fsub_rn(s[t][e], safe)), p1 = ex2(__fsub_rn(s[t][e + 2], safe));
          l[t][e] = __fmaf_rn(l[t][e], alpha[t][e], __fadd_rn(p0, p1));
          // the weights enter the second product as bf16 (relative error 2^-9 each, against the
          // output's own bf16 rounding of the same size); their sum l keeps all 32 bits
          sm.p[n][16 * warp + oct] = f2bf(p0);
          sm.p[n][16 * warp + oct + 8] = f2bf(p1);
        }
      // V of the next tile goes where this tile's K was
      if (j_next < k_end) load(slot, c.v, r_next);
      cp_async_commit();
      const int j_after = j_next < k_end ? next_tile(j_next + kTile) : j_next;
      const long long r_after = j_after < k_end ? key_row(j_after) : -1;
      cp_async_wait<2>();
      __syncthreads();  // V and the weights have landed
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x][t][e] = __fmul_rn(o[x][t][e], alpha[t][e & 1]);
      const uint32_t vbase = smem_u32(sm.kv[sv]);
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k) {
        uint32_t pf[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          pf[t][0] = *reinterpret_cast<const uint32_t*>(&sm.p[8 * t + oct][16 * k + 2 * quad]);
          pf[t][1] = *reinterpret_cast<const uint32_t*>(&sm.p[8 * t + oct][16 * k + 8 + 2 * quad]);
        }
        const int row = 16 * k + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          uint32_t vf[4];
          const int ch = (warp * MT + x) * 2 + ((lane >> 3) & 1);
          ldsm_x4_t(vf, vbase + row * Dh * 2 + ((ch ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_bf16(o[x][t], vf, pf[t][0], pf[t][1]);
        }
      }
      j = j_next;
      j_next = j_after;
      r_next = r_after;
      slot = sk2;
    }
    cp_async_wait_all();
    // sums over the key lanes and warps; is the numerator finite?
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= !isfinite(o[x][t][e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[t][e];
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) x = __fadd_rn(x, __shfl_xor_sync(0xFFFFFFFFu, x, d));
        if (oct == 0) sm.sum[warp][8 * t + 2 * quad + e] = x;
      }
    }
    odd = __syncthreads_or(odd);
    const bool whole = sl.count == 1;  // the only slab: finish here
    const long long part = (long long)b * a.max_slabs + i_slab;
    auto store = [&](int r, int d, float val, float ll) {
      const int s = r / a.G, h = kh * a.G + r - s * a.G;
      if (whole) {
        const long long t = b * a.S + s;
        float y = ll == 0.0f ? 0.0f : __fdiv_rn(val, ll);
        if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[t * a.gate_ld + h * a.gate_hs + d])));
        a.out[(t * a.nq + h) * Dh + d] = f2bf(y);
      } else {
        a.ws_o[((part * a.S + s) * a.nq + h) * Dh + d] = val;
      }
    };
    if (!odd) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = 8 * t + 2 * quad + e, r = row0 + n;
          if (r >= R) continue;
          const float ll = __fadd_rn(__fadd_rn(sm.sum[0][n], sm.sum[1][n]), __fadd_rn(sm.sum[2][n], sm.sum[3][n]));
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            const int d = (warp * MT + x) * 16 + oct;
            store(r, d, o[x][t][e], ll);
            store(r, d + 8, o[x][t][e + 2], ll);
          }
          if (!whole && warp == 0 && oct == 0) {
            const int s = r / a.G;
            a.ws_ml[(part * a.S + s) * a.nq + kh * a.G + r - s * a.G] = make_float2(m[t][e], ll);
          }
        }
    } else {
      // An infinity or NaN reached a sum: from a key that the row sees, or, as 0 * inf, from one it does not.
      // Settle it by the definition, a warp per row, reading visible keys only.
      for (int n = warp; n < 8 * NT && row0 + n < R; n += 4) {
        const int r = row0 + n, s = r / a.G, h = kh * a.G + r - s * a.G;
        float mm = -INFINITY, ll = 0.0f, oo[Dh / 32] = {};
        attend_row_strict<Dh>(c, a.q + (long long)(b * a.S + s) * a.q_ld + (long long)h * Dh, b, kh, pos0 + s, k_begin,
                              k_end, a.vis, a.scale2, a.err, mm, ll, oo);
        for (int e = 0; e < Dh / 32; ++e) store(r, lane * (Dh / 32) + e, oo[e], ll);
        if (!whole && lane == 0) a.ws_ml[(part * a.S + s) * a.nq + h] = make_float2(mm, ll);
      }
    }
    __syncthreads();  // the shared buffers are free for the next unit
  }
}

// Joins the slabs of one (row, 64 dims): M = max m_i, o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.  256
// threads: 16 lanes of 4 dims x 16 groups, group g taking the slabs whose number is g mod 16, the groups'
// sums added in order, so the order of additions belongs to the slabs' positions.
template <int Dh>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedView c, DecodeArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ float s_m[8];
  __shared__ float4 s_o[16][16];
  __shared__ float s_l[16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = tid >> 4, d_blk = (blockIdx.x % (Dh / 64)) * 64;
  const int d = d_blk + (tid & 15) * 4, br = blockIdx.x / (Dh / 64);
  const int rows = a.S * a.nq, b = br / rows, r = br - b * rows;  // r = s * nq + h
  const SlabList sl = slab_list(c, a, b, nullptr);
  if (sl.count == 1) return;
  const float2* ml = a.ws_ml + (long long)b * a.max_slabs * rows + r;
  const float* po = a.ws_o + ((long long)b * a.max_slabs * rows + r) * Dh + d;
  float M = -INFINITY;
  for (int i = tid; i < sl.count; i += 256) M = fmaxf(M, ml[(long long)i * rows].x);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, x));
  if (lane == 0) s_m[warp] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) M = fmaxf(M, s_m[i]);
  const float safe = M == -INFINITY ? 0.0f : M;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.0f;
  // listed slab i has number i (i < first) or from + i - first: begin each group at its residue
  auto walk = [&](int i0, int i1, int shift) {
    int i = i0 + ((g - (i0 + shift)) & 15);
#pragma unroll 4
    for (; i < i1; i += 16) {
      const float2 v = ml[(long long)i * rows];
      const float4 x = *reinterpret_cast<const float4*>(po + (long long)i * rows * Dh);
      const float w = ex2(__fsub_rn(v.x, safe));
      den = __fmaf_rn(w, v.y, den);
      if (w != 0.0f) {  // a slab this row sees nothing of adds nothing
        acc.x = __fmaf_rn(w, x.x, acc.x);
        acc.y = __fmaf_rn(w, x.y, acc.y);
        acc.z = __fmaf_rn(w, x.z, acc.z);
        acc.w = __fmaf_rn(w, x.w, acc.w);
      }
    }
  };
  walk(0, sl.first, 0);
  walk(sl.first, sl.count, sl.from - sl.first);
  s_o[g][tid & 15] = acc;
  if ((tid & 15) == 0) s_l[g] = den;
  __syncthreads();
  if (tid >= 64) return;
  const float* so = reinterpret_cast<const float*>(s_o);
  float y = 0.0f, ll = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    y = __fadd_rn(y, so[i * 64 + tid]);
    ll = __fadd_rn(ll, s_l[i]);
  }
  y = ll == 0.0f ? 0.0f : __fdiv_rn(y, ll);
  const int s = r / a.nq, h = r - s * a.nq, dd = d_blk + tid;
  const long long t = b * a.S + s;
  if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[t * a.gate_ld + h * a.gate_hs + dd])));
  a.out[(t * a.nq + h) * Dh + dd] = f2bf(y);
}

// ----------------------------------------------------------------------------- host
int paged_view(const qmtp_paged_cache* c, PagedView* v) {
  if (!c || !c->k || !c->v || !c->table || !c->lens) return QMTP_ERR_ARG;
  if (c->B < 1 || c->B > kMaxSeqs || c->n_kv < 1 || c->pages < 1 || c->table_w < 1 || c->ld_table < c->table_w)
    return QMTP_ERR_SHAPE;
  if (c->Dh != 64 && c->Dh != 128 && c->Dh != 256) return QMTP_ERR_UNSUPPORTED;
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) return QMTP_ERR_UNSUPPORTED;
  if (c->pages > (1ll << 31) / c->page / c->n_kv - 1 || c->table_w > (1 << 30) / c->page) return QMTP_ERR_SHAPE;
  if (!aligned16(c->k) || !aligned16(c->v)) return QMTP_ERR_ALIGN;
  int lg = 4;
  while ((1 << lg) < c->page) ++lg;
  *v = PagedView{static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->table, c->lens, c->pages,
                 c->ld_table, c->n_kv, lg, c->table_w, c->B};
  return QMTP_OK;
}

int paged_check_args(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  if (!a || !a->q || !a->out) return QMTP_ERR_ARG;
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale) || a->window < 0 || a->sinks < 0) return QMTP_ERR_ARG;
  if (a->T < 1 || a->n_q < 1 || a->n_q % c->n_kv) return QMTP_ERR_SHAPE;
  if (a->n_q / c->n_kv > 64) return QMTP_ERR_UNSUPPORTED;
  if (a->q_ld % 8 || (a->q_ld && a->q_ld < (long long)a->n_q * c->Dh)) return QMTP_ERR_SHAPE;
  if (a->gate && (a->gate_ld % 8 || a->gate_hs % 8)) return QMTP_ERR_SHAPE;
  if (!aligned16(a->q) || !aligned16(a->out) || (a->gate && !aligned16(a->gate))) return QMTP_ERR_ALIGN;
  return QMTP_OK;
}

static bool fine_slabs(int window) { return window > 0 && window <= kFineKeys; }

// Most slabs that one sequence can list: all of its table, or sinks and window with their ragged ends.
static int max_slabs(const qmtp_paged_args* a, const qmtp_paged_cache* c, int S) {
  const bool fine = fine_slabs(a->window);
  const long long cap = (long long)c->table_w * c->page;
  long long n = slab_of(int(cap - 1), fine) + 1;
  if (a->window > 0) {
    const long long k = fine ? kFineSlab : 1;  // fine slabs only: a wide window may cover every slab
    if (fine) n = std::min(n, (std::min<long long>(a->sinks, cap) + k - 1) / k + (a->window + S + k - 1) / k + 1);
  }
  return int(n);
}

static size_t align_up(size_t x) { return (x + 255) & ~size_t(255); }

template <int Dh, int NT>
static int launch_decode(const PagedView& v, const DecodeArgs& a, long long units, cudaStream_t st) {
  const size_t smem = sizeof(DecodeSmem<Dh, NT>) + (v.B + 1) * sizeof(int);
  static DeviceOnce ready;
  if (!ready([] {
        return cudaFuncSetAttribute(paged_decode_kernel<Dh, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(sizeof(DecodeSmem<Dh, NT>) + (kMaxSeqs + 1) * sizeof(int)));
      }))
    return QMTP_ERR_CUDA;
  const int per_sm = Dh == 256 ? 2 : 4;
  const int grid = int(std::min<long long>(units, (long long)sm_count() * per_sm));
  launch_kernel(paged_decode_kernel<Dh, NT>, dim3(grid), dim3(128), smem, st, v, a);
  if (a.max_slabs > 1)
    launch_kernel(paged_join_kernel<Dh>, dim3(v.B * a.S * a.nq * (Dh / 64)), dim3(256), 0, st, v, a);
  return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
}

template <int Dh>
static int launch_append(const PagedView& v, const AppendArgs& a, cudaStream_t st) {
  const int per = kAppendSteps * (32 / (Dh / 8));
  const long long warps = (long long)a.T * ((a.nq + 2 * v.nkv + per - 1) / per);
  launch_kernel(paged_append_kernel<Dh>, dim3(unsigned((warps + 7) / 8)), dim3(256), 0, st, v, a);
  return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
}

}  // namespace qmtp

using namespace qmtp;

extern "C" int qmtp_paged_append(const void* qkv, long long ld, int T, const int* cu, int n_q, int gated,
                                 const void* q_w, const void* k_w, float eps, const float* cos_t, const float* sin_t,
                                 int rotary, int max_pos, void* q_out, const qmtp_paged_cache* cache, void* stream) {
  PagedView v;
  if (const int rc = paged_view(cache, &v)) return rc;
  if (!qkv || !q_out || (cos_t == nullptr) != (sin_t == nullptr) || !(eps >= 0.0f)) return QMTP_ERR_ARG;
  if (T < 1 || n_q < 1 || ld % 8 || ld < (long long)(n_q * (gated ? 2 : 1) + 2 * cache->n_kv) * cache->Dh)
    return QMTP_ERR_SHAPE;
  if (!cu && T % cache->B) return QMTP_ERR_SHAPE;
  if (cos_t && (rotary < 16 || rotary > cache->Dh || rotary % 16)) return QMTP_ERR_UNSUPPORTED;
  if (cos_t && max_pos < 1) return QMTP_ERR_SHAPE;
  for (const void* p : {qkv, q_w, k_w, (const void*)cos_t, (const void*)sin_t, (const void*)q_out})
    if (p && !aligned16(p)) return QMTP_ERR_ALIGN;
  if ((long long)T * (n_q + 2 * cache->n_kv) >= (1ll << 33)) return QMTP_ERR_SHAPE;  // the grid stays below 2^31
  unsigned* err = device_error_ptr();
  if (!err) return QMTP_ERR_CUDA;
  AppendArgs a{static_cast<const uint16_t*>(qkv), ld, cu, static_cast<const uint16_t*>(q_w),
               static_cast<const uint16_t*>(k_w), cos_t, sin_t, static_cast<uint16_t*>(q_out), eps, T,
               cu ? 0 : T / cache->B, n_q, gated ? 1 : 0, cos_t ? rotary : 0, max_pos, err};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->Dh == 64 ? launch_append<64>(v, a, st)
                         : cache->Dh == 128 ? launch_append<128>(v, a, st) : launch_append<256>(v, a, st);
}

extern "C" size_t qmtp_paged_attention_workspace(const qmtp_paged_args* args, const qmtp_paged_cache* cache) {
  if (!args || !cache || cache->B < 1 || cache->table_w < 1 || cache->page < 1) return 0;
  const int S = args->T / cache->B, n = max_slabs(args, cache, S);
  if (n <= 1) return 0;
  const size_t rows = size_t(cache->B) * n * S * args->n_q;
  return align_up(rows * cache->Dh * sizeof(float)) + rows * sizeof(float2);
}

extern "C" int qmtp_paged_attention(const qmtp_paged_args* args, const qmtp_paged_cache* cache, void* workspace,
                                    size_t ws_bytes, void* stream) {
  PagedView v;
  if (const int rc = paged_view(cache, &v)) return rc;
  if (const int rc = paged_check_args(args, cache)) return rc;
  if (args->T % v.B) return QMTP_ERR_SHAPE;
  const int S = args->T / v.B, G = args->n_q / v.nkv;
  if (S > kMaxS) return QMTP_ERR_UNSUPPORTED;
  const size_t need = qmtp_paged_attention_workspace(args, cache);
  if (need && !workspace) return QMTP_ERR_ARG;
  if (ws_bytes < need) return QMTP_ERR_SHAPE;
  if (need && !aligned16(workspace)) return QMTP_ERR_ALIGN;
  unsigned* err = device_error_ptr();
  if (!err) return QMTP_ERR_CUDA;
  DecodeArgs a{};
  a.q = static_cast<const uint16_t*>(args->q);
  a.gate = static_cast<const uint16_t*>(args->gate);
  a.out = static_cast<uint16_t*>(args->out);
  a.q_ld = args->q_ld ? args->q_ld : (long long)args->n_q * cache->Dh;
  a.gate_ld = args->gate_ld;
  a.gate_hs = args->gate_hs;
  a.nq = args->n_q;
  a.S = S;
  a.G = G;
  a.scale2 = args->scale * kLog2e;
  a.vis = Visible{args->window, args->sinks};
  a.fine = fine_slabs(args->window);
  a.max_slabs = max_slabs(args, cache, S);
  a.err = err;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) +
                                      align_up(size_t(v.B) * a.max_slabs * S * a.nq * cache->Dh * sizeof(float)));
  const bool two = S * G > 8;
  a.row_tiles = (S * G + (two ? 15 : 7)) / (two ? 16 : 8);
  const long long units = (long long)v.B * a.max_slabs * v.nkv * a.row_tiles;
  if (units >= (1ll << 31) || (long long)v.B * S * a.nq >= (1ll << 28)) return QMTP_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define QMTP_DECODE(D) (two ? launch_decode<D, 2>(v, a, units, st) : launch_decode<D, 1>(v, a, units, st))
  return cache->Dh == 64 ? QMTP_DECODE(64) : cache->Dh == 128 ? QMTP_DECODE(128) : QMTP_DECODE(256);
#undef QMTP_DECODE
}
