// Paged key/value cache: the writer (per-head q/k norm + rotation + append) and the attention of the
// newest tokens, split over the cache's length and joined.  The prompt form is in paged_prompt.cu.
#include <algorithm>
#include <cmath>

#include <cuda_bf16.h>

#include "paged.cuh"

namespace qmtp {

// ----------------------------------------------------------------------------- append
// Per head row x of q or k: y = x / sqrt(mean x^2 + eps) * w, then dims (i, i + R/2), i < R/2, turn by the
// position's angle: (y_i c - y_j s, y_j c + y_i s).  All fp32; one rounding to bf16 on the way out.
// A group of Dh / 8 lanes owns a row.  Of the rotated dims a lane takes four and their four partners (two loads of
// 8 bytes), so a pair never leaves its lane; of the others, eight in a row.  A warp takes STEPS steps of
// 32 / (Dh / 8) head rows of one token, loads them all first and shares the token's angles.  Bound: HBM (one read,
// one write), with the instructions close behind: an early form with 285 a row step took 129 us for 15437 tokens,
// where this takes 73 (5.3 TB/s).
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

template <int Dh, int STEPS, bool LOOP>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedView c, AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int LPR = Dh / 8, RPS = 32 / LPR;  // lanes per row, rows per step
  const int lane = threadIdx.x & 31, sub = lane % LPR, half = a.rotary / 2;
  const bool turns = 8 * sub < a.rotary;
  const int da = turns ? 4 * sub : 8 * sub, db = turns ? half + 4 * sub : 8 * sub + 4;  // this lane's dims: 4 from each on
  const unsigned heads = a.nq + 2 * c.nkv, units = (heads + STEPS * RPS - 1) / (STEPS * RPS);  // warps per token
  const unsigned wid = blockIdx.x * 8 + (threadIdx.x >> 5);
  // LOOP: a warp takes a whole token, the next step's rows under way; else one step
  const int t = LOOP ? wid : wid / units;
  int h0 = (LOOP ? 0 : wid - t * units) * STEPS * RPS + lane / LPR;
  if (t >= a.T) return;
  const uint16_t* row = a.qkv + (long long)t * a.ld;
  uint2 x[STEPS][2], ahead[LOOP ? STEPS : 1][2];
  auto fetch = [&](uint2 (*to)[2], int first) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = first + i * RPS;
      to[i][0] = to[i][1] = make_uint2(0, 0);
      if (h < int(heads)) {
        const uint16_t* src = row + (a.gated ? (h < a.nq ? 2 * h : a.nq + h) : h) * Dh;
        to[i][0] = *reinterpret_cast<const uint2*>(src + da);
        to[i][1] = *reinterpret_cast<const uint2*>(src + db);
      }
    }
  };
  fetch(x, h0);
  // the row's sequence and position
  int b, p;
  if (a.cu == nullptr) {
    b = t / a.S;
    p = seq_len(c, b, a.err) - a.S + (t - b * a.S);
  } else {
    // the sequence [cu[b], cu[b + 1]) that holds row t, a warp's worth at a time; offsets that are none hold no row
    b = p = -1;
    bool bad = false;
    for (int i = 0; i < c.B; i += 32) {
      const int k = i + lane, c0 = k < c.B ? a.cu[k] : 0, c1 = k < c.B ? a.cu[k + 1] : 0;
      const bool good = c0 >= 0 && c0 <= c1 && c1 <= a.T;
      bad |= !good;
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, good && c0 <= t && t < c1);
      if (hit && b < 0) {
        b = i + __ffs(hit) - 1;
        p = t - __shfl_sync(0xFFFFFFFFu, c1, __ffs(hit) - 1);
      }
    }
    if (bad) atomicOr(a.err, DEVERR_BADARG);
    if (b < 0) return;  // a row of no sequence
    p += seq_len(c, b, a.err);
  }
  if (p < 0) return;
  const bool far = a.cos_t != nullptr && p >= a.max_pos;
  if (far || (p >> c.page_log) >= c.table_w) {
    if (lane == 0) atomicOr(a.err, DEVERR_BADARG);
    return;
  }
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turns) {
    cs = *reinterpret_cast<const float4*>(a.cos_t + (long long)p * half + da);
    sn = *reinterpret_cast<const float4*>(a.sin_t + (long long)p * half + da);
  }
  const uint64_t c2[2] = {f2_pack(cs.x, cs.y), f2_pack(cs.z, cs.w)};
  const uint64_t s2[2] = {f2_pack(sn.x, sn.y), f2_pack(sn.z, sn.w)}, n2[2] = {f2_pack(-sn.x, -sn.y), f2_pack(-sn.z, -sn.w)};
  const long long r0 = cache_row(c, b, 0, p, a.err);  // the position's row of key head 0; a head is a page further
  for (unsigned u = 0; u < (LOOP ? units : 1u); ++u) {
    if (LOOP && u + 1 < units) fetch(ahead, h0 + STEPS * RPS);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = h0 + i * RPS;
      const bool live = h < int(heads), isq = h < a.nq, isv = h >= a.nq + c.nkv;
      uint2 out[2] = {x[i][0], x[i][1]};
      const uint16_t* weight = isq ? a.qw : a.kw;
      if (__any_sync(0xFFFFFFFFu, live && !isv)) {  // values are copied as they are
        uint64_t y[2][2];
        uint64_t ss2 = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          y[k][0] = f2_pack(bflo(x[i][k].x), bfhi(x[i][k].x));
          y[k][1] = f2_pack(bflo(x[i][k].y), bfhi(x[i][k].y));
          ss2 = f2_fma(y[k][0], y[k][0], ss2);
          ss2 = f2_fma(y[k][1], y[k][1], ss2);
        }
        if (a.qw != nullptr || a.kw != nullptr) {  // the sum by every lane: a step may hold rows with and without a norm
          float sa, sb;
          f2_unpack(ss2, sa, sb);
          float ss = __fadd_rn(sa, sb);
#pragma unroll
          for (int d = LPR / 2; d >= 1; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, d));
          const float r = rsqrtf(__fmaf_rn(ss, 1.0f / Dh, a.eps));
          const uint64_t r2 = f2_pack(r, r);
          if (weight != nullptr) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint2 w = *reinterpret_cast<const uint2*>(weight + (k ? db : da));
              y[k][0] = f2_mul(f2_mul(y[k][0], r2), f2_pack(bflo(w.x), bfhi(w.x)));
              y[k][1] = f2_mul(f2_mul(y[k][1], r2), f2_pack(bflo(w.y), bfhi(w.y)));
            }
          }
        }
        if (turns) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint64_t u = y[0][k], v = y[1][k];
            y[0][k] = f2_fma(u, c2[k], f2_mul(v, n2[k]));
            y[1][k] = f2_fma(v, c2[k], f2_mul(u, s2[k]));
          }
        }
        if (!isv) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float e[4];
            f2_unpack(y[k][0], e[0], e[1]);
            f2_unpack(y[k][1], e[2], e[3]);
            out[k] = make_uint2(pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]));
          }
        }
      }
      uint16_t* dst = nullptr;
      if (live && isq)
        dst = a.q_out + ((long long)t * a.nq + h) * Dh;
      else if (live && r0 >= 0)
        dst = (isv ? c.v : c.k) + (r0 + ((long long)(isv ? h - a.nq - c.nkv : h - a.nq) << c.page_log)) * Dh;
      if (dst) {
        *reinterpret_cast<uint2*>(dst + da) = out[0];
        *reinterpret_cast<uint2*>(dst + db) = out[1];
      }
    }
    if (LOOP) {
      h0 += STEPS * RPS;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        x[i][0] = ahead[LOOP ? i : 0][0];
        x[i][1] = ahead[LOOP ? i : 0][1];
      }
    }
  }
}

// ----------------------------------------------------------------------------- decode attention
// A unit of work is (sequence, slab of keys, key head, tile of query rows); rows are the S tokens x G query
// heads of the key head.  Scores and the weighted sum run on the tensor cores with the keys (dims) on the
// M side, S^T = K Q^T and O^T = V^T P^T (m16n8k16), so a group of 4 or 8 rows fills the 8-wide N side.
// The keys' bytes bound it (4 flops a byte and row group), so mma.sync is enough: its pipe is a small part of the
// time the bytes take.  A CTA takes units u, u + grid, ...; its producer warp walks their tiles ahead of the four
// consumer warps and keeps the ring full across units, so neither a unit's first load nor its table
// lookups are waited for.
constexpr int kFineKeys = 4096;
constexpr int kSlabLog = 9;
constexpr int kMaxS = 8;

// Slabs have fixed positions: [0, 4096) in fine slabs, then slabs of 512; fine ones everywhere for windows up to 4096.
// Fine slabs spread a short context over the SMs: 128, 256 or 512 keys, so that the key heads of 4096 keys make
// 128 units or more; larger ones keep the partial results (Dh + 2 floats a row and slab) small next to the keys.
// Fixed positions make a row's arithmetic independent of the batch and of the call's other rows.
struct Slabs {
  int fine_log;
  int all_fine;
  __host__ __device__ __forceinline__ int of(int j) const {
    return all_fine || j < kFineKeys ? j >> fine_log : (kFineKeys >> fine_log) + ((j - kFineKeys) >> kSlabLog);
  }
  __device__ __forceinline__ int begin(int i) const {
    const int n = kFineKeys >> fine_log;
    return all_fine || i <= n ? i << fine_log : kFineKeys + ((i - n) << kSlabLog);
  }
};

struct DecodeArgs {
  const uint16_t *q, *gate;
  uint16_t* out;
  long long q_ld, gate_ld, gate_hs;
  float* ws_o;    // [B][max_slabs][S * nq][Dh] numerators
  float2* ws_ml;  // [B][max_slabs][S * nq] running maximum (base 2) and sum
  int nq, S, G, row_tiles, max_slabs;
  Slabs slabs;
  int one_round;   // no CTA has a second unit
  int cluster;     // FUSED: CTAs of a cluster
  unsigned inv_g;  // ceil(2^16 / G): r / G = r * inv_g >> 16 for r < 512, G <= 64
  float scale2;   // scale * log2(e)
  Visible vis;
  unsigned* err;
};

// Slabs of one sequence that some query row of it sees: [0, first) and [from, from + count - first).
struct SlabList {
  int lo, first, from, count;
};
__device__ __forceinline__ SlabList slab_list(const DecodeArgs& a, int len) {
  SlabList s;
  s.lo = a.vis.first(max(0, len - a.S));  // the first key of the oldest row's window
  s.from = a.slabs.of(s.lo);
  s.first = a.vis.sinks > 0 && s.lo > 0 ? min(a.slabs.of(min(a.vis.sinks, s.lo) - 1) + 1, s.from) : 0;
  s.count = len > 0 ? s.first + a.slabs.of(len - 1) + 1 - s.from : 1;  // an empty sequence: one empty slab
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
// Barrier of the four consumer warps.
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// NT: groups of 8 query rows in a tile (1, 2 or 4).  A step takes TK keys, 16 KG a warp for the scores; small heads take
// more of them, which spreads a step's waits and barriers over more work.
template <int Dh, int NT>
struct DecodeCfg {
  static constexpr int KG = Dh == 64 ? 2 : 1, TK = 64 * KG;
  static constexpr int per_sm = Dh == 256 || (NT == 4 && Dh == 128) ? 2 : 3;
  static constexpr int ring = Dh == 256 ? 3 : NT < 4 ? 4 : Dh == 128 ? 6 : 3;  // entries: a tile of K or of V each
};

template <int Dh, int NT>
struct DecodeSmem {
  using Cfg = DecodeCfg<Dh, NT>;
  uint16_t kv[Cfg::ring][Cfg::TK * Dh];  // 64-dim column blocks of 128-byte swizzled rows
  static constexpr int QS = NT > 1 ? 1 : 2;  // per_sm CTAs have to fit on an SM
  uint16_t q[QS][8 * NT][Dh + 8];
  __nv_bfloat16 p[8 * NT][Cfg::TK + 8];  // weights, [row][key]
  float mx[4][8 * NT];
  float sum[2][4][8 * NT];
  float2 ml[8 * NT];  // FUSED: this slab's maxima and sums
  uint64_t full[Cfg::ring], empty[Cfg::ring], q_full[2], q_empty[2];
  int bad[2];
  int scan[8];
  WaitState wait;
};

__device__ __forceinline__ float join_weight(float m, float M) { return m == -INFINITY ? 0.0f : ex2(__fsub_rn(m, M)); }
// Four dims of a finished row: sum / denominator (0 where the row sees no key; 0 / 0 = NaN where every score that it sees
// is -inf), the gate, one rounding.
__device__ __forceinline__ void join_store(const DecodeArgs& a, float (&y)[4], float ll, bool sees, uint2 gate, uint16_t* dst) {
  const float g[4] = {bflo(gate.x), bfhi(gate.x), bflo(gate.y), bfhi(gate.y)};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    y[k] = sees ? __fdiv_rn(y[k], ll) : 0.0f;
    if (a.gate) y[k] = __fmul_rn(y[k], sigmoid_f32(g[k]));
  }
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
}

struct DecodeUnit {
  int b, kh, row0, len, lo, k_begin, k_end, part;
};

// Unit u of the call: s_pre the slabs before every sequence, s_len their lengths.  Not inlined: the producer and the
// consumers call it once a unit, and the kernel's code is fetched anew for every launch.
__device__ __noinline__ DecodeUnit decode_unit(const int* s_pre, const int* s_len, const DecodeArgs& a, int B, int nkv,
                                               int rows, int u) {
  DecodeUnit x;
  const int per = nkv * a.row_tiles, slab_g = u / per, rest = u - slab_g * per;
  x.kh = rest / a.row_tiles;
  x.row0 = (rest - x.kh * a.row_tiles) * rows;
  int b = 0;  // the last sequence that begins at or before this slab
  for (int step = 1 << (31 - __clz(B)); step > 0; step >>= 1)
    if (b + step < B && s_pre[b + step] <= slab_g) b += step;
  x.b = b;
  x.len = s_len[b];
  const SlabList sl = slab_list(a, x.len);
  x.lo = sl.lo;
  x.part = slab_g - s_pre[b];
  const int slab = x.part < sl.first ? x.part : sl.from + x.part - sl.first;
  x.k_begin = a.slabs.begin(slab);
  x.k_end = min(a.slabs.begin(slab + 1), x.len);
  return x;
}

// FUSED: one launch for short tables.  The slabs of a (sequence, key head, row tile) are the CTAs of a cluster, one unit
// each; their partial results stay in shared memory and every CTA joins its share of the rows' dims through
// distributed shared memory, in the join kernels' order.
template <int Dh, int NT, bool FUSED>
__global__ void __launch_bounds__(160, DecodeCfg<Dh, NT>::per_sm)
paged_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, PagedView c,
                    const __grid_constant__ DecodeArgs a) {
  if (FUSED || a.one_round) pdl_trigger();  // otherwise when the last unit is done: a waiting successor's blocks take up room
  extern __shared__ uint8_t smem_raw[];
  using Smem = DecodeSmem<Dh, NT>;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  int* s_pre = reinterpret_cast<int*>(&sm + 1);  // [B + 1] slabs before sequence b
  int* s_len = s_pre + c.B + 1;                  // [B]
  using Cfg = DecodeCfg<Dh, NT>;
  constexpr int RING = Cfg::ring, CB = Dh / 64, QS = Smem::QS, KG = Cfg::KG, kTile = Cfg::TK;
  constexpr int MT = Dh / 64;  // 16-dim tiles of a warp in the weighted sum
  constexpr float kNone = -INFINITY;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 128) {
    for (int i = 0; i < RING; ++i) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 4); }
    for (int i = 0; i < 2; ++i) { mbar_init(&sm.q_full[i], 1); mbar_init(&sm.q_empty[i], 4); sm.bad[i] = 0; }
    sm.wait = WaitState{0, 0};
    fence_mbar_init();
  }
  pdl_wait();
  const int R = a.S * a.G, per = c.nkv * a.row_tiles;
  int units = 1;
  DecodeUnit mine;      // FUSED: the CTA's unit
  SlabList mine_slabs;
  if (FUSED) {
    const int rank = cluster_rank(), cl = blockIdx.x / a.cluster, rest = cl % per;
    mine.b = cl / per;
    mine.kh = rest / a.row_tiles;
    mine.row0 = (rest - mine.kh * a.row_tiles) * 8 * NT;
    mine.len = seq_len(c, mine.b, rank == 0 ? a.err : nullptr);
    mine_slabs = slab_list(a, mine.len);
    mine.lo = mine_slabs.lo;
    mine.part = rank;
    const int slab = rank < mine_slabs.first ? rank : mine_slabs.from + rank - mine_slabs.first;
    mine.k_begin = rank < mine_slabs.count ? a.slabs.begin(slab) : 0;
    mine.k_end = rank < mine_slabs.count ? min(a.slabs.begin(slab + 1), mine.len) : 0;
  } else {
    int total = 0;
    for (int b0 = 0; b0 < c.B; b0 += 160) {
      const int b = b0 + tid;
      int n = 0, len = 0;
      if (b < c.B) {
        len = seq_len(c, b, blockIdx.x == 0 ? a.err : nullptr);
        n = slab_list(a, len).count;
      }
      int chunk;
      const int before = block_excl_scan(n, sm.scan, chunk);
      if (b < c.B) { s_pre[b] = total + before; s_len[b] = len; }
      total += chunk;
    }
    if (tid == 0) s_pre[c.B] = total;
    units = total * per;
  }
  __syncthreads();
  const int u0 = FUSED ? 0 : blockIdx.x, ustep = FUSED ? 1 : gridDim.x;
  auto unit_at = [&](int u) { return FUSED ? mine : decode_unit(s_pre, s_len, a, c.B, c.nkv, 8 * NT, u); };
  // the next tile of the unit, from key j on, that holds a needed key
  auto next_tile = [&](const DecodeUnit& x, int j) {
    while (j < x.k_end && a.vis.window != 0 && j + kTile <= x.lo && j >= a.vis.sinks) j += kTile;
    return j;
  };

  if (warp == 4) {
    // -------------------------------------------------------------------- producer
    const int box = min(1 << c.page_log, kTile), parts = kTile / box;
    const long long none = (c.pages * c.nkv) << c.page_log;  // past the end: reads as zeros
    // cache row of part `lane` of the tile at key j; a page that no row needs is not looked at
    auto part_row = [&](const DecodeUnit& x, int j) -> int {
      const int key = j + lane * box;
      if (lane >= parts || key >= x.k_end || (a.vis.window != 0 && key + box <= x.lo && key >= a.vis.sinks))
        return int(none);
      const long long r = cache_row(c, x.b, x.kh, key, a.err);
      return int(r < 0 ? none : r);
    };
    const int part = lane / CB, cb = lane - part * CB;
    int e = 0, uq = 0;
    auto load = [&](const CUtensorMap* map, int row) {
      const int st = e % RING;
      if (!warp_wait(&sm.wait, &sm.empty[st], ((e / RING) & 1) ^ 1, a.err)) return;
      if (lane == 0) mbar_expect_tx(&sm.full[st], kTile * Dh * 2);
      __syncwarp();
      const int r = __shfl_sync(0xFFFFFFFFu, row, min(part, parts - 1));
      if (part < parts)
        tma_load_2d(reinterpret_cast<uint8_t*>(sm.kv[st]) + cb * kTile * 128 + part * box * 128, map, cb * 64, r,
                    &sm.full[st], policy_evict_first());
      ++e;
    };
    DecodeUnit x;
    int j = 0, row = 0, u = u0;
    if (u < units) {
      x = unit_at(u);
      j = next_tile(x, x.k_begin);
      if (j < x.k_end) row = part_row(x, j);
    }
    bool head = true;
    while (u < units && !given_up(&sm.wait)) {
      // the tile after this one, its table entries on their way while this one's copies are issued
      DecodeUnit xn = x;
      int un = u, jn = j < x.k_end ? next_tile(x, j + kTile) : x.k_end;
      if (jn >= x.k_end) {
        un = u + ustep;
        if (un < units) {
          xn = unit_at(un);
          jn = next_tile(xn, xn.k_begin);
        }
      }
      const int row_n = un < units && jn < xn.k_end ? part_row(xn, jn) : 0;
      if (j < x.k_end) {
        load(&tk, row);
        load(&tv, row);
      }
      if (head) {  // the unit's query rows (their place may still be in use: behind the first copies)
        const int st = uq % QS, rows = min(8 * NT, R - x.row0);
        if (!warp_wait(&sm.wait, &sm.q_empty[st], ((uq / QS) & 1) ^ 1, a.err)) break;
        if (lane == 0) mbar_expect_tx(&sm.q_full[st], rows * Dh * 2);
        __syncwarp();
        if (lane < rows) {
          const int r = x.row0 + lane, s = r * a.inv_g >> 16;
          bulk_g2s(sm.q[st][lane], a.q + (long long)(x.b * a.S + s) * a.q_ld + (long long)(x.kh * a.G + r - s * a.G) * Dh,
                   Dh * 2, &sm.q_full[st], policy_evict_last());
        }
        ++uq;
      }
      head = un != u;
      x = xn;
      u = un;
      j = jn;
      row = row_n;
    }
    if (given_up(&sm.wait)) {  // copies in flight end before the CTA does
      for (int i = max(0, e - RING); i < e; ++i) mbar_wait_bounded(&sm.full[i % RING], (i / RING) & 1, a.err, 1u << 22);
      for (int i = max(0, uq - QS); i < uq; ++i) mbar_wait_bounded(&sm.q_full[i % QS], (i / QS) & 1, a.err, 1u << 22);
    }
    if (!FUSED) return;
    __syncwarp();
  }

  // ---------------------------------------------------------------------- consumers
  const int quad = lane & 3, oct = lane >> 2;
  int e = 0, uq = 0;
  for (int u = warp == 4 ? units : u0; u < units; u += ustep, ++uq) {
    const DecodeUnit x = unit_at(u);
    const int pos0 = x.len - a.S, set = uq & 1;
    int prow[NT][2];  // positions of this lane's rows n = 8 t + 2 quad + i
    float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = x.row0 + 8 * t + 2 * quad + i;
        prow[t][i] = r < R ? pos0 + int(r * a.inv_g >> 16) : -1;
        m[t][i] = kNone;
        l[t][i] = 0.0f;
      }
#pragma unroll
      for (int y = 0; y < MT; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[y][t][i] = 0.0f;
    }
    warp_wait(&sm.wait, &sm.q_full[uq % QS], (uq / QS) & 1, a.err);
    const uint32_t qbase = smem_u32(sm.q[uq % QS]) + (lane & 7) * (Dh + 8) * 2 + (lane >> 3) * 16;
    for (int j = next_tile(x, x.k_begin); j < x.k_end; j = next_tile(x, j + kTile)) {
      const int sk = e % RING, sv = (e + 1) % RING;
      warp_wait(&sm.wait, &sm.full[sk], (e / RING) & 1, a.err);
      float s[KG][NT][4];
#pragma unroll
      for (int g = 0; g < KG; ++g)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[g][t][i] = 0.0f;
      {
        const int row = 16 * KG * warp + (lane & 15);
        const uint32_t base = smem_u32(sm.kv[sk]) + row * 128;
#pragma unroll
        for (int k = 0; k < Dh / 32; ++k) {  // 32 dims: two K fragments a key group, one load of query fragments a row group
          uint32_t k0[KG][4], k1[KG][4];
          const uint32_t cbase = base + (k >> 1) * kTile * 128;
          const int ch = (k & 1) * 4 + (lane >> 4);
#pragma unroll
          for (int g = 0; g < KG; ++g) {
            ldsm_x4(k0[g], cbase + g * 16 * 128 + ((ch ^ (row & 7)) << 4));
            ldsm_x4(k1[g], cbase + g * 16 * 128 + (((ch + 2) ^ (row & 7)) << 4));
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t qf[4];
            ldsm_x4(qf, qbase + t * 8 * (Dh + 8) * 2 + k * 64);
#pragma unroll
            for (int g = 0; g < KG; ++g) {
              mma_bf16(s[g][t], k0[g], qf[0], qf[1]);
              mma_bf16(s[g][t], k1[g], qf[2], qf[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[sk]);
      if (j + kTile - 1 > pos0 || (a.vis.window != 0 && j < a.vis.first(x.len - 1))) {  // not every row sees every key
#pragma unroll
        for (int g = 0; g < KG; ++g)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!a.vis(prow[t][i & 1], j + 16 * KG * warp + 16 * g + oct + 8 * (i >> 1))) s[g][t][i] = kNone;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = fmaxf(s[0][t][i], s[0][t][i + 2]);
#pragma unroll
          for (int g = 1; g < KG; ++g) v = fmaxf(v, fmaxf(s[g][t][i], s[g][t][i + 2]));
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
          if (oct == 0) sm.mx[warp][8 * t + 2 * quad + i] = v;
        }
      consumers_sync();
      float alpha[NT][2];
      bool grown = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = 8 * t + 2 * quad + i;
          const float top = fmaxf(fmaxf(sm.mx[0][n], sm.mx[1][n]), fmaxf(sm.mx[2][n], sm.mx[3][n]));
          const float mn = fmaxf(m[t][i], __fmul_rn(top, a.scale2));
          const float neg = mn == kNone ? 0.0f : -mn;  // nothing seen yet: every weight is 0
          alpha[t][i] = ex2(__fadd_rn(m[t][i], neg));
          grown |= mn != m[t][i];
          m[t][i] = mn;
          float sum = 0.0f;
#pragma unroll
          for (int g = 0; g < KG; ++g) {
            const float p0 = ex2(__fmaf_rn(s[g][t][i], a.scale2, neg)), p1 = ex2(__fmaf_rn(s[g][t][i + 2], a.scale2, neg));
            sum = __fadd_rn(sum, __fadd_rn(p0, p1));
            // the weights enter the second product as bf16 (off by at most 2^-8 relative each, as the output's own
            // rounding is); their sum l keeps all 32 bits
            sm.p[n][16 * KG * warp + 16 * g + oct] = __float2bfloat16_rn(p0);
            sm.p[n][16 * KG * warp + 16 * g + oct + 8] = __float2bfloat16_rn(p1);
          }
          l[t][i] = __fmaf_rn(l[t][i], alpha[t][i], sum);
        }
      warp_wait(&sm.wait, &sm.full[sv], ((e + 1) / RING) & 1, a.err);
      if (j + kTile > x.len || (a.vis.window != 0 && j < x.lo)) {
        // values that no row sees may be anything, and their weight 0 has to stay 0: cleared
        uint8_t* v = reinterpret_cast<uint8_t*>(sm.kv[sv]);
        for (int i = tid; i < CB * kTile * 8; i += 128) {
          const int key = j + ((i >> 3) & (kTile - 1));
          if (key >= x.len || (a.vis.window != 0 && key < x.lo && key >= a.vis.sinks))
            *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
      }
      consumers_sync();
      if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
        for (int y = 0; y < MT; ++y)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[y][t][i] = __fmul_rn(o[y][t][i], alpha[t][i & 1]);
      }
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
        for (int y = 0; y < MT; ++y) {
          uint32_t vf[4];
          const int ch = (warp * MT + y) * 2 + ((lane >> 3) & 1);
          ldsm_x4_t(vf, vbase + (ch >> 3) * kTile * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_bf16(o[y][t], vf, pf[t][0], pf[t][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[sv]);
      e += 2;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.q_empty[uq % QS]);
    if (!FUSED && u + ustep >= units) pdl_trigger();
    // sums over the key lanes and warps; is the numerator finite?
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = l[t][i];
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
        if (oct == 0) sm.sum[set][warp][8 * t + 2 * quad + i] = v;
        bool odd = false;
#pragma unroll
        for (int y = 0; y < MT; ++y) odd |= !isfinite(o[y][t][i]) || !isfinite(o[y][t][i + 2]);
        if (odd && x.row0 + 8 * t + 2 * quad + i < R) sm.bad[set] = 1;
      }
    consumers_sync();
    const bool odd = sm.bad[set] != 0;
    if (tid == 0) sm.bad[set ^ 1] = 0;
    const long long part = ((long long)x.b * a.max_slabs + x.part) * a.S;
    if (!odd) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = 8 * t + 2 * quad + i, r = x.row0 + n, s = r * a.inv_g >> 16;
          if (r >= R) continue;
          const long long at = FUSED ? n : (part + s) * a.nq + x.kh * a.G + r - s * a.G;
          float* dst = (FUSED ? reinterpret_cast<float*>(sm.kv) : a.ws_o) + at * Dh + warp * MT * 16 + oct;
#pragma unroll
          for (int y = 0; y < MT; ++y) {
            dst[16 * y] = o[y][t][i];
            dst[16 * y + 8] = o[y][t][i + 2];
          }
          if (warp == 0 && oct == 0)
            (FUSED ? sm.ml : a.ws_ml)[at] = make_float2(m[t][i], __fadd_rn(__fadd_rn(sm.sum[set][0][n], sm.sum[set][1][n]),
                                                         __fadd_rn(sm.sum[set][2][n], sm.sum[set][3][n])));
        }
      __syncwarp();
    } else {
      // An infinity or NaN reached a sum: from a key that the row sees, or, as 0 * inf, from one it does not.
      // Settle it by the definition, a warp per row, reading visible keys only.
      for (int n = warp; n < 8 * NT && x.row0 + n < R; n += 4) {
        const int r = x.row0 + n, s = r * a.inv_g >> 16, h = x.kh * a.G + r - s * a.G;
        float mm = kNone, ll = 0.0f, oo[Dh / 32] = {};
        attend_row_strict<Dh>(c, a.q + (long long)(x.b * a.S + s) * a.q_ld + (long long)h * Dh, x.b, x.kh, pos0 + s,
                              x.k_begin, x.k_end, a.vis, a.scale2, a.err, mm, ll, oo);
        const long long at = FUSED ? n : (part + s) * a.nq + h;
        float* dst = (FUSED ? reinterpret_cast<float*>(sm.kv) : a.ws_o) + at * Dh;
        for (int i = 0; i < Dh / 32; ++i) dst[lane * (Dh / 32) + i] = oo[i];
        if (lane == 0) (FUSED ? sm.ml : a.ws_ml)[at] = make_float2(mm, ll);
        sign_of_life(&sm.wait);
      }
    }
  }
  if (FUSED) {
    __syncwarp();
    cluster_sync_all();  // every slab's numerators and (maximum, sum) can be read
    const int rows = min(8 * NT, R - mine.row0), n_parts = mine_slabs.count;
    for (int i = mine.part * 160 + tid; i < rows * (Dh / 4); i += a.cluster * 160) {
      const int n = i / (Dh / 4), d = (i - n * (Dh / 4)) * 4;
      const int r = mine.row0 + n, s = r * a.inv_g >> 16, h = mine.kh * a.G + r - s * a.G;
      const long long t = mine.b * a.S + s;
      uint2 g2 = make_uint2(0, 0);
      if (a.gate) g2 = *reinterpret_cast<const uint2*>(a.gate + t * a.gate_ld + h * a.gate_hs + d);
      const float* mlp = reinterpret_cast<const float*>(&sm.ml[n]);
      const float* op = reinterpret_cast<const float*>(sm.kv) + n * Dh + d;
      // class k: slab number k of the first ones (few calls have any), and the one of the others with that residue
      float m1[16], l1[16];
      int part_of[16];
      float M = kNone;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int pt = mine_slabs.first + ((k - mine_slabs.from) & 15);
        part_of[k] = pt < n_parts ? pt : 0;
        m1[k] = ld_dsmem(mlp, part_of[k]);
        l1[k] = ld_dsmem(mlp + 1, part_of[k]);
        if (pt >= n_parts) m1[k] = kNone;
        M = fmaxf(M, m1[k]);
      }
      for (int k = 0; k < mine_slabs.first; ++k) M = fmaxf(M, ld_dsmem(mlp, k));
      float y[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.0f;
#pragma unroll
      for (int k0 = 0; k0 < 16; k0 += 8) {
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = ld_dsmem_v4(op, part_of[k0 + k]);
          // a class without a slab adds nothing, whatever the slab read in its place holds: 0 times an infinity would be NaN
          if (mine_slabs.first + ((k0 + k - mine_slabs.from) & 15) >= n_parts) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float z[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.0f;
          if (k0 + k < mine_slabs.first) {
            const float w = join_weight(ld_dsmem(mlp, k0 + k), M);
            const float4 u = ld_dsmem_v4(op, k0 + k);
            den = __fmaf_rn(w, ld_dsmem(mlp + 1, k0 + k), den);
            z[0] = __fmaf_rn(w, u.x, z[0]);
            z[1] = __fmaf_rn(w, u.y, z[1]);
            z[2] = __fmaf_rn(w, u.z, z[2]);
            z[3] = __fmaf_rn(w, u.w, z[3]);
          }
          const float w = join_weight(m1[k0 + k], M);
          den = __fmaf_rn(w, l1[k0 + k], den);
          y[0] = __fadd_rn(y[0], __fmaf_rn(w, v[k].x, z[0]));
          y[1] = __fadd_rn(y[1], __fmaf_rn(w, v[k].y, z[1]));
          y[2] = __fadd_rn(y[2], __fmaf_rn(w, v[k].z, z[2]));
          y[3] = __fadd_rn(y[3], __fmaf_rn(w, v[k].w, z[3]));
          ll = __fadd_rn(ll, den);
        }
      }
      join_store(a, y, ll, mine.len - a.S + s >= 0, g2, a.out + (t * a.nq + h) * Dh + d);
    }
    __syncwarp();
    cluster_sync_all();  // the others have read this CTA's shared memory
  }
}

// Joins a row's slabs: M = max m_i, o = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i, the gate, the rounding.  A slab's class
// is its number mod 16; every class is summed in rising order, then the classes in order, so the order of
// additions belongs to the slabs' positions, however they are dealt to threads.  Two ways to deal them:
//   wide (few rows): a block per (row, 64 dims), 16 threads of 4 dims for each class;
//   warp (many rows): a warp per (row, 128 dims), 4 dims a lane and every class in its registers, no barrier; four blocks
//   an SM (24 x 3 tokens, window 1024: 32.3 us, with 137 registers and three blocks 34.5).
struct JoinRow {
  const float2* ml;   // slab i at ml[i * stride]
  const float* o;     // ... at o[i * stride * Dh]
  long long out, gate, stride;
  SlabList sl;
  bool sees;  // the row's position is one of the sequence, so it sees at least its own key
};
template <int Dh>
__device__ __forceinline__ JoinRow join_row(const PagedView& c, const DecodeArgs& a, int br) {
  JoinRow j;
  const int rows = a.S * a.nq, b = br / rows, r = br - b * rows, s = r / a.nq, h = r - s * a.nq;
  const int len = seq_len(c, b, nullptr);
  j.sl = slab_list(a, len);
  j.sees = len - a.S + s >= 0;
  j.ml = a.ws_ml + (long long)b * a.max_slabs * rows + r;
  j.o = a.ws_o + ((long long)b * a.max_slabs * rows + r) * Dh;
  j.stride = rows;
  const long long t = b * a.S + s;
  j.out = (t * a.nq + h) * Dh;
  j.gate = t * a.gate_ld + h * a.gate_hs;
  return j;
}

template <int Dh>
__global__ void __launch_bounds__(256) paged_join_wide_kernel(PagedView c, DecodeArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ float s_m[8];
  __shared__ float4 s_o[16][16];
  __shared__ float s_l[16];
  const int tid = threadIdx.x, lane = tid & 31, cls = tid >> 4, d0 = blockIdx.x % (Dh / 64) * 64;
  const JoinRow j = join_row<Dh>(c, a, blockIdx.x / (Dh / 64));
  float gate = 0.0f;
  if (a.gate && tid < 64) gate = bf2f(a.gate[j.gate + d0 + tid]);
  float M = -INFINITY;
  for (int i = tid; i < j.sl.count; i += 256) M = fmaxf(M, j.ml[i * j.stride].x);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, x));
  if (lane == 0) s_m[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) M = fmaxf(M, s_m[i]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.0f;
  const float* po = j.o + d0 + 4 * (tid & 15);
  // listed slab i has number i (i < first) or from + i - first: a class begins at its residue
  for (int part = 0; part < 2; ++part) {
    const int i0 = part ? j.sl.first : 0, i1 = part ? j.sl.count : j.sl.first, number0 = part ? j.sl.from : 0;
#pragma unroll 16
    for (int i = i0 + ((cls - number0) & 15); i < i1; i += 16) {
      const float2 v = j.ml[i * j.stride];
      const float4 x = *reinterpret_cast<const float4*>(po + i * j.stride * Dh);
      const float w = join_weight(v.x, M);
      den = __fmaf_rn(w, v.y, den);
      acc.x = __fmaf_rn(w, x.x, acc.x);
      acc.y = __fmaf_rn(w, x.y, acc.y);
      acc.z = __fmaf_rn(w, x.z, acc.z);
      acc.w = __fmaf_rn(w, x.w, acc.w);
    }
  }
  s_o[cls][tid & 15] = acc;
  if ((tid & 15) == 0) s_l[cls] = den;
  __syncthreads();
  if (tid >= 64) return;
  const float* so = reinterpret_cast<const float*>(s_o);
  float y = 0.0f, ll = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    y = __fadd_rn(y, so[i * 64 + tid]);
    ll = __fadd_rn(ll, s_l[i]);
  }
  y = j.sees ? __fdiv_rn(y, ll) : 0.0f;
  if (a.gate) y = __fmul_rn(y, sigmoid_f32(gate));
  a.out[j.out + d0 + tid] = f2bf(y);
}

template <int Dh>
__global__ void __launch_bounds__(128, 4) paged_join_warp_kernel(PagedView c, DecodeArgs a) {
  pdl_wait();
  constexpr int LPR = Dh / 4, RPW = LPR < 32 ? 32 / LPR : 1, WPR = LPR > 32 ? LPR / 32 : 1;  // lanes a row, rows a warp
  const int lane = threadIdx.x & 31, wid = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int br = wid / WPR * RPW + (RPW > 1 ? lane / LPR : 0), d = RPW > 1 ? lane % LPR * 4 : (wid % WPR * 32 + lane) * 4;
  const bool live = br < c.B * a.S * a.nq;
  const JoinRow j = join_row<Dh>(c, a, live ? br : 0);
  uint2 g2 = make_uint2(0, 0);
  if (a.gate) g2 = *reinterpret_cast<const uint2*>(a.gate + j.gate + d);
  // half-warp lane k looks after class k: its slabs' weights and its share of the denominator
  const int k0 = lane & 15, half = lane & 16;
  float M = -INFINITY, den = 0.0f;
  for (int i = k0; i < j.sl.count; i += 16) M = fmaxf(M, j.ml[i * j.stride].x);
#pragma unroll
  for (int x = 8; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, x));
  const long long step = j.stride * Dh;
  float4 acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    // slabs i0 .. i1 of the list have numbers number0 ..: sixteen numbers, one of each class, at a time
    const int i0 = part ? j.sl.first : 0, i1 = part ? j.sl.count : j.sl.first, number0 = part ? j.sl.from : 0;
#pragma unroll 1
    for (int i = i0 - (number0 & 15); __any_sync(0xFFFFFFFFu, i < i1); i += 16) {
      float w = 0.0f;
      if (i + k0 >= i0 && i + k0 < i1) {
        const float2 v = j.ml[(i + k0) * j.stride];
        w = join_weight(v.x, M);
        den = __fmaf_rn(w, v.y, den);
      }
      const float* po = j.o + d;
#pragma unroll
      for (int h = 0; h < 16; h += 8) {
        float4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)  // eight loads under way at once; numbers outside the list read a listed slab
          x[k] = *reinterpret_cast<const float4*>(po + min(max(i + h + k, 0), j.sl.count - 1) * step);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float wk = __shfl_sync(0xFFFFFFFFu, w, half + h + k);
          if (i + h + k >= i0 && i + h + k < i1) {  // ... and add nothing: 0 times an infinity would be NaN
            acc[h + k].x = __fmaf_rn(wk, x[k].x, acc[h + k].x);
            acc[h + k].y = __fmaf_rn(wk, x[k].y, acc[h + k].y);
            acc[h + k].z = __fmaf_rn(wk, x[k].z, acc[h + k].z);
            acc[h + k].w = __fmaf_rn(wk, x[k].w, acc[h + k].w);
          }
        }
      }
    }
  }
  float y[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    y[0] = __fadd_rn(y[0], acc[k].x);
    y[1] = __fadd_rn(y[1], acc[k].y);
    y[2] = __fadd_rn(y[2], acc[k].z);
    y[3] = __fadd_rn(y[3], acc[k].w);
    ll = __fadd_rn(ll, __shfl_sync(0xFFFFFFFFu, den, half + k));
  }
  if (live) join_store(a, y, ll, j.sees, g2, a.out + j.out + d);
}

// ----------------------------------------------------------------------------- host
int paged_view(const qmtp_paged_cache* c, PagedView* v) {
  if (!c || !c->k || !c->v || !c->table || !c->lens) return QMTP_ERR_ARG;
  if (c->B < 1 || c->B > kMaxSeqs || c->n_kv < 1 || c->n_kv > kMaxHeads || c->pages < 1 || c->table_w < 1 || c->ld_table < c->table_w)
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
  if (!(a->scale > 0.0f) || !std::isfinite(a->scale * kLog2e) || a->window < 0 || a->sinks < 0) return QMTP_ERR_ARG;
  if (a->T < 1 || a->n_q < 1 || a->n_q > kMaxHeads || a->n_q % c->n_kv) return QMTP_ERR_SHAPE;
  if (a->n_q / c->n_kv > 64) return QMTP_ERR_UNSUPPORTED;
  if (a->q_ld % 8 || (a->q_ld && a->q_ld < (long long)a->n_q * c->Dh)) return QMTP_ERR_SHAPE;
  if (a->gate && (a->gate_ld % 8 || a->gate_hs % 8)) return QMTP_ERR_SHAPE;
  if (!aligned16(a->q) || !aligned16(a->out) || (a->gate && !aligned16(a->gate))) return QMTP_ERR_ALIGN;
  return QMTP_OK;
}

static Slabs slabs_for(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  return Slabs{c->n_kv < 8 ? 7 : c->n_kv < 16 ? 8 : 9, a->window > 0 && a->window <= kFineKeys};
}

// Most slabs that one sequence can list: all of its table, or sinks and window with their ragged ends.
static int max_slabs(const qmtp_paged_args* a, const qmtp_paged_cache* c, int S) {
  const Slabs sl = slabs_for(a, c);
  const long long cap = (long long)c->table_w * c->page, k = 1ll << sl.fine_log;
  long long n = sl.of(int(cap - 1)) + 1;
  if (sl.all_fine) n = std::min(n, (std::min<long long>(a->sinks, cap) + k - 1) / k + (a->window + S + k - 1) / k + 1);
  return int(n);
}

// Rows of a tile, in groups of 8: as many as there are up to 32, at 256 dims up to 16 (registers); K and V are read
// once a tile.
static int row_groups(int rows, int Dh) { return rows <= 8 ? 1 : rows <= 16 || Dh == 256 ? 2 : 4; }

// CTAs of a cluster when the call fits the fused form, else 0: a table of at most 16 slabs, and clusters that fill no
// more than one CTA per SM.  Measured (4 key heads of 256, 4 rows): 515 keys 7.7 us fused, 8.7 with the
// join as a second launch.
static int fused_cluster(const qmtp_paged_args* a, const qmtp_paged_cache* c, int S) {
  const int n = max_slabs(a, c, S), rows = S * (a->n_q / c->n_kv), per_tile = 8 * row_groups(rows, c->Dh);
  const int cluster = n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16;
  return n <= 16 && (long long)c->B * c->n_kv * ((rows + per_tile - 1) / per_tile) * cluster <= sm_count() ? cluster : 0;
}

static size_t align_up(size_t x) { return (x + 255) & ~size_t(255); }

template <int Dh, int NT>
static int launch_decode(const PagedView& v, DecodeArgs a, long long units, cudaStream_t st) {
  constexpr size_t fixed = sizeof(DecodeSmem<Dh, NT>) + 1024;
  static DeviceOnce ready;
  if (!ready([] {
        if (const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<Dh, NT, false>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       int(fixed + (2 * kMaxSeqs + 1) * sizeof(int))))
          return e;
        if (const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<Dh, NT, true>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, int(fixed)))
          return e;
        return cudaFuncSetAttribute(paged_decode_kernel<Dh, NT, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      }))
    return QMTP_ERR_CUDA;
  CUtensorMap tk, tv;
  const cuuint64_t kd[2] = {Dh, cuuint64_t((v.pages * v.nkv) << v.page_log)}, ks[1] = {Dh * 2};
  const cuuint32_t kb[2] = {64, cuuint32_t(std::min(1 << v.page_log, DecodeCfg<Dh, NT>::TK))};
  if (!encode_pages(&tk, v.k, 2, kd, ks, kb) || !encode_pages(&tv, v.v, 2, kd, ks, kb)) return QMTP_ERR_CUDA;
  if (a.cluster) {
    const int grid = v.B * v.nkv * a.row_tiles * a.cluster;
    launch_kernel_cluster(paged_decode_kernel<Dh, NT, true>, dim3(grid), dim3(160), fixed, st, a.cluster, tk, tv, v, a);
    return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
  }
  const int grid = int(std::min<long long>(units, (long long)sm_count() * DecodeCfg<Dh, NT>::per_sm));
  a.one_round = grid == units;
  launch_kernel(paged_decode_kernel<Dh, NT, false>, dim3(grid), dim3(160), fixed + (2 * v.B + 1) * sizeof(int), st, tk, tv, v,
                a);
  const int rows = v.B * a.S * a.nq;
  if (rows >= 2 * sm_count()) {
    constexpr int RPW = Dh == 64 ? 2 : 1, WPR = Dh == 256 ? 2 : 1;
    launch_kernel(paged_join_warp_kernel<Dh>, dim3((((rows + RPW - 1) / RPW) * WPR + 3) / 4), dim3(128), 0, st, v, a);
  } else {
    launch_kernel(paged_join_wide_kernel<Dh>, dim3(rows * (Dh / 64)), dim3(256), 0, st, v, a);
  }
  return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
}

template <int Dh, int STEPS, bool LOOP>
static int launch_append_steps(const PagedView& v, const AppendArgs& a, cudaStream_t st) {
  const int per = STEPS * (32 / (Dh / 8));
  const long long warps = LOOP ? a.T : (long long)a.T * ((a.nq + 2 * v.nkv + per - 1) / per);
  launch_kernel(paged_append_kernel<Dh, STEPS, LOOP>, dim3(unsigned((warps + 7) / 8)), dim3(256), 0, st, v, a);
  return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
}

// Few rows: one a lane group, so that none waits for another (3 tokens of 16 + 8 heads of 256: 2.2 us, with four steps a
// warp 3.5; 200 tokens 3.6 and 4.1).  More: four steps a warp, which share a token's position and angles (2048 tokens:
// 11.3 us, with one step 17.1, by whole tokens 16.3).  With 64 tokens an SM and more, whole tokens (15437: 73 us, with four
// steps 78).
template <int Dh>
static int launch_append(const PagedView& v, const AppendArgs& a, cudaStream_t st) {
  const long long groups = (long long)a.T * (a.nq + 2 * v.nkv) * Dh / 256;  // warps of one row step
  if (groups < 32ll * sm_count()) return launch_append_steps<Dh, 1, false>(v, a, st);
  if (a.T < 64 * sm_count()) return launch_append_steps<Dh, 4, false>(v, a, st);
  return launch_append_steps<Dh, 3, true>(v, a, st);
}

}  // namespace qmtp

using namespace qmtp;

extern "C" int qmtp_paged_append(const void* qkv, long long ld, int T, const int* cu, int n_q, int gated,
                                 const void* q_w, const void* k_w, float eps, const float* cos_t, const float* sin_t,
                                 int rotary, int max_pos, void* q_out, const qmtp_paged_cache* cache, void* stream) {
  PagedView v;
  if (const int rc = paged_view(cache, &v)) return rc;
  if (!qkv || !q_out || (cos_t == nullptr) != (sin_t == nullptr) || !(eps >= 0.0f)) return QMTP_ERR_ARG;
  if (T < 1 || n_q < 1 || n_q > kMaxHeads || ld % 8 || ld < (long long)(n_q * (gated ? 2 : 1) + 2 * cache->n_kv) * cache->Dh)
    return QMTP_ERR_SHAPE;
  if (!cu && T % cache->B) return QMTP_ERR_SHAPE;
  if (cos_t && (rotary < 16 || rotary > cache->Dh || rotary % 16)) return QMTP_ERR_UNSUPPORTED;
  if (cos_t && max_pos < 1) return QMTP_ERR_SHAPE;
  for (const void* p : {qkv, q_w, k_w, (const void*)cos_t, (const void*)sin_t, (const void*)q_out})
    if (p && !aligned16(p)) return QMTP_ERR_ALIGN;
  if ((long long)T * (n_q + 2 * cache->n_kv) >= (1ll << 31)) return QMTP_ERR_SHAPE;  // warps are counted in 32 bits
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
  PagedView v;
  if (paged_view(cache, &v) || paged_check_args(args, cache)) return 0;
  const int S = args->T / cache->B, n = max_slabs(args, cache, S);
  if (fused_cluster(args, cache, S)) return 0;
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
  a.inv_g = (65536 + G - 1) / G;
  a.scale2 = args->scale * kLog2e;
  a.vis = Visible{args->window, args->sinks};
  a.slabs = slabs_for(args, cache);
  a.max_slabs = max_slabs(args, cache, S);
  a.cluster = fused_cluster(args, cache, S);
  a.err = err;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) +
                                      align_up(size_t(v.B) * a.max_slabs * S * a.nq * cache->Dh * sizeof(float)));
  const int nt = row_groups(S * G, cache->Dh);
  a.row_tiles = (S * G + 8 * nt - 1) / (8 * nt);
  const long long units = (long long)v.B * a.max_slabs * v.nkv * a.row_tiles;
  if (units >= (1ll << 30) || (long long)v.B * S * a.nq >= (1ll << 28)) return QMTP_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define QMTP_DECODE(D) (nt == 1 ? launch_decode<D, 1>(v, a, units, st) : launch_decode<D, 2>(v, a, units, st))
  if (cache->Dh == 256) return QMTP_DECODE(256);
  if (nt == 4) return cache->Dh == 64 ? launch_decode<64, 4>(v, a, units, st) : launch_decode<128, 4>(v, a, units, st);
  return cache->Dh == 64 ? QMTP_DECODE(64) : QMTP_DECODE(128);
#undef QMTP_DECODE
}
