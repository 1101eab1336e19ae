// Prompt attention over the paged cache on the tensor cores (tcgen05), for a ragged batch of chunks.
//
// A CTA owns NQ tiles of 128 query rows (128 / G tokens x the G query heads of a key head: all of them read
// the same keys) and walks the key tiles (128 keys) they see with the running maximum m and sum l of the
// softmax.  Per key tile: S = Q K^T into TMEM; the tile's 128 threads, one row each, turn S into weights
// P = 2^(S scale2 - m) in place (bf16); O += P V with P from TMEM.  O stays in TMEM and is rescaled only
// when a row's maximum has grown by more than 2^kSlack since the last rescale, which leaves P <= 2^kSlack;
// the final division by l takes it out again.
//   warps 0 .. 4 NQ - 1   softmax, and at the end O / l, the gate and the store
//   warp 4 NQ             TMA: pages into a ring of tiles (128-byte swizzle)
//   warp 4 NQ + 1         MMA issue
// Dh 256: one row tile, two S buffers (the scores of the next key tile run under this tile's softmax).
// Dh 128, 64: two row tiles of one S buffer each, which take turns.  TMEM: O in columns [0, 256), S in [256, 512).
#include <algorithm>

#include "paged.cuh"

namespace qmtp {

constexpr int kRows = 128;  // query rows of a tile
constexpr int kKeys = 128;  // keys of a tile
constexpr float kSlack = 8.0f;

template <int Dh>
struct PromptCfg {
  static constexpr int NQ = Dh == 256 ? 1 : 2;               // row tiles per CTA
  static constexpr int E = Dh == 256 ? 2 : 1;                // ring entries per K or V tile (halves of 32 KB)
  static constexpr int entry = kKeys * Dh * 2 / E;           // bytes
  static constexpr int stages = Dh == 64 ? 8 : 5;
  static constexpr int threads = NQ * 128 + 64;
  static constexpr unsigned poly = Dh == 256 ? 0x22 : 0x52;  // of every 8 pairs of exponentials, those done by ex2_poly
  static constexpr int q_bytes = kRows * Dh * 2;
  static constexpr int smem = NQ * q_bytes + stages * entry + 1024 + 512;
};

struct PromptArgs {
  const int* cu;
  const uint16_t *q, *gate;
  uint16_t* out;
  long long q_ld, gate_ld, gate_hs;
  float* ws_o;    // [splits][T][nq][Dh]
  float2* ws_ml;  // [splits][T][nq]
  int T, nq, G, tpt, splits;  // tpt: tokens per row tile
  float scale2;
  Visible vis;
  unsigned* err;
};

struct PromptBars {
  uint64_t full[8], empty[8], q_full, s_full[2], p_full[2][2];
  uint64_t pv[2];    // a phase per key tile but the last: O holds the products up to it
  uint64_t done[2];  // the last product
  uint32_t tmem;
  int dead;   // a wait ran out: every later wait returns at once
  int b, tile, n, c0, len;  // this CTA's sequence, row tile, new tokens, first row, length
};

// 128-byte swizzled operand tile: rows of 128 bytes in groups of 8 (1024 bytes).  K-major (Q, K): `sbo` is the group
// stride, lbo unused; MN-major (V): lbo is the distance of the next 64 dims, sbo that of the next 8 keys.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t((lbo >> 4) & 0x3FFFu) << 16) |
         (uint64_t((sbo >> 4) & 0x3FFFu) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
// The loaded registers may be used from here on: the wait, tied to them so that no use moves above it.
__device__ __forceinline__ void tmem_ld32_ready(float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]),
                 "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]),
                 "+r"(u[16]), "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]),
                 "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])::"memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x != 0;
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^f on [-1/2, 1/2], degree 4: least squares at Chebyshev points, reweighted until the relative error was level, 2^-18.5
constexpr float kE0 = 0.9999993f, kE1 = 0.6931218f, kE2 = 0.24024744f, kE3 = 0.05591786f, kE4 = 0.009570101f;
// 2^x of a pair without the exponential unit, x <= 8; below 2^-126, and at -inf, 0.  x = n + f, |f| <= 1/2, by adding and
// taking away 1.5 2^23; 2^f by the polynomial, n into the exponent bits.
__device__ __forceinline__ void ex2_poly(uint64_t v, float& p0, float& p1) {
  const uint64_t magic = f2_pack(12582912.0f, 12582912.0f), unmagic = f2_pack(-12582912.0f, -12582912.0f);
  const uint64_t minus = f2_pack(-1.0f, -1.0f);
  const uint64_t r = f2_add(v, magic);
  const uint64_t f = f2_fma(f2_add(r, unmagic), minus, v);
  uint64_t p = f2_fma(f2_pack(kE4, kE4), f, f2_pack(kE3, kE3));
  p = f2_fma(p, f, f2_pack(kE2, kE2));
  p = f2_fma(p, f, f2_pack(kE1, kE1));
  p = f2_fma(p, f, f2_pack(kE0, kE0));
  float x0, x1, r0, r1;
  f2_unpack(v, x0, x1);
  f2_unpack(r, r0, r1);
  f2_unpack(p, p0, p1);
  p0 = x0 < -126.0f ? 0.0f : __int_as_float(__float_as_int(p0) + (__float_as_int(r0) << 23));
  p1 = x1 < -126.0f ? 0.0f : __int_as_float(__float_as_int(p1) + (__float_as_int(r1) << 23));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <int Dh>
__global__ void __launch_bounds__(PromptCfg<Dh>::threads, 1)
paged_prompt_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, PagedView c, PromptArgs a) {
  using Cfg = PromptCfg<Dh>;
  constexpr int NQ = Cfg::NQ, E = Cfg::E, NS = Cfg::stages, CB = Dh / 64;  // CB: 64-dim column blocks
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* s_q = base;
  uint8_t* s_ring = base + NQ * Cfg::q_bytes;
  PromptBars* bars = reinterpret_cast<PromptBars*>(s_ring + NS * Cfg::entry);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kh = blockIdx.x % c.nkv, item = blockIdx.x / c.nkv, split = blockIdx.y;
  const int TT = NQ * a.tpt;  // tokens per CTA

  if (warp == 4 * NQ + 1) tmem_alloc(&bars->tmem, 512);
  if (warp == 4 * NQ && lane == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], 1); }
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i][0], 128);
      mbar_init(&bars->p_full[i][1], 128);
      mbar_init(&bars->pv[i], 1);
      mbar_init(&bars->done[i], 1);
    }
    bars->dead = 0;
    fence_mbar_init();
  }
  pdl_wait();
  if (warp == 0) {  // which sequence and row tile: the sequences' tiles counted a warp at a time
    if (lane == 0) bars->b = -1;
    __syncwarp();
    int before = 0;
    for (int i = 0; i < c.B; i += 32) {
      const int k = i + lane;
      int n = 0, c0 = 0;
      if (k < c.B) {
        c0 = a.cu[k];
        const int c1 = a.cu[k + 1];
        n = c1 - c0;
        if (c0 < 0 || c1 > a.T || c1 < c0) {
          if (blockIdx.x == 0) atomicOr(a.err, DEVERR_BADARG);
          n = 0;
        }
      }
      const int tiles = (n + TT - 1) / TT;
      int incl = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += x;
      }
      const int at = item - before - (incl - tiles);
      if (at >= 0 && at < tiles) {
        bars->b = k;
        bars->tile = tiles - 1 - at;  // the last rows see the most keys: first
        bars->n = n;
        bars->c0 = c0;
        bars->len = seq_len(c, k, a.err);
      }
      before += __shfl_sync(0xFFFFFFFFu, incl, 31);
      if (item < before) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const int b = bars->b;
  if (b >= 0) {
    const int n = bars->n, len = bars->len, c0 = bars->c0, tok0 = bars->tile * TT;
    const int p_first = len - n + tok0, p_last = len - n + min(n, tok0 + TT) - 1;
    const int chains = NQ == 1 || tok0 + a.tpt >= n ? 1 : 2;  // row tiles that hold a token
    // key tiles: [0, sink_tiles), then [lo / 128, p_last / 128]
    const int lo = a.vis.first(max(p_first, 0)), lo_tile = lo / kKeys;
    const int sink_tiles =
        a.vis.sinks > 0 && lo > 0 ? min((min(a.vis.sinks, lo) + kKeys - 1) / kKeys, lo_tile) : 0;
    const int nt_all = p_last < 0 ? 0 : sink_tiles + p_last / kKeys + 1 - lo_tile;
    const int t_begin = int((long long)nt_all * split / a.splits), t_end = int((long long)nt_all * (split + 1) / a.splits);
    const int nt = t_end - t_begin;
    auto tile_key = [&](int t) {  // first key of the t-th tile of this CTA
      t += t_begin;
      return (t < sink_tiles ? t : lo_tile + t - sink_tiles) * kKeys;
    };
    // ring position of K(t), V(t): Dh 256 loads K0 K1 V0 K2 V1 ..., otherwise K0 V0 K1 V1 ...
    auto pos_k = [&](int t) { return NQ == 1 ? (t == 0 ? 0 : 2 * t - 1) : 2 * t; };
    auto pos_v = [&](int t) { return NQ == 1 ? min(2 * t + 2, 2 * nt - 1) : 2 * t + 1; };

    if (warp == 4 * NQ) {
      // ------------------------------------------------------------------ TMA
      const int box = min(1 << c.page_log, kKeys / E), parts = kKeys / box;  // rows per box, boxes down a tile
      const long long none = (c.pages * c.nkv) << c.page_log;                // past the end: reads as zeros
      // cache row of part `lane` of the tile at key j (a page that no row needs is not looked at)
      auto part_row = [&](int j) -> int {
        const int key = j + lane * box;
        if (lane >= parts || key > p_last || (a.vis.window != 0 && key + box <= lo && key >= a.vis.sinks))
          return int(none);
        const long long r = cache_row(c, b, kh, key, a.err);
        return int(r < 0 ? none : r);
      };
      int issued = 0;
      auto load = [&](const CUtensorMap* map, int pos, bool is_v, int row) {
#pragma unroll
        for (int h = 0; h < E; ++h) {
          const int e = pos * E + h, st = e % NS;
          bar_wait(&bars->dead, &bars->empty[st], ((e / NS) & 1) ^ 1, a.err);
          if (*reinterpret_cast<volatile int*>(&bars->dead)) return;
          if (lane == 0) mbar_expect_tx(&bars->full[st], Cfg::entry);
          __syncwarp();
          issued = e + 1;
          uint8_t* dst = s_ring + st * Cfg::entry;
          // an entry: K all keys x half the dims, V half the keys x all dims (E == 2), else the whole tile
          const int ncb = is_v ? CB : CB / E, np = is_v ? parts / E : parts, rows = is_v ? kKeys / E : kKeys;
          const int part = lane / ncb, cb = lane - part * ncb;
          const int r = __shfl_sync(0xFFFFFFFFu, row, (is_v ? h * np : 0) + min(part, np - 1));
          if (part < np)
            tma_load_2d(dst + cb * rows * 128 + part * box * 128, map, (is_v ? cb : h * ncb + cb) * 64, r, &bars->full[st],
                        policy_evict_last());
        }
      };
      if (nt > 0) {
        if (lane == 0) mbar_expect_tx(&bars->q_full, uint32_t(chains) * a.G * a.tpt * Dh * 2);
        __syncwarp();
        if (lane < chains * CB) {
          const int w = lane / CB, cb = lane - w * CB;
          tma_load_3d(s_q + w * Cfg::q_bytes + cb * kRows * 128, &tq, cb * 64, kh * a.G, c0 + tok0 + w * a.tpt, &bars->q_full);
        }
        int row = part_row(tile_key(0)), row_next = nt > 1 ? part_row(tile_key(1)) : 0;
        load(&tk, pos_k(0), false, row);
        for (int t = 0; t < nt; ++t) {
          const int row_after = t + 2 < nt ? part_row(tile_key(t + 2)) : 0;
          if (NQ == 2) load(&tv, pos_v(t), true, row);
          if (t + 1 < nt) load(&tk, pos_k(t + 1), false, row_next);
          if (NQ == 1) load(&tv, pos_v(t), true, row);
          row = row_next;
          row_next = row_after;
        }
        if (*reinterpret_cast<volatile int*>(&bars->dead)) {  // copies in flight end before the CTA does
          mbar_wait_bounded(&bars->q_full, 0, a.err, 1u << 22);
          for (int e = max(0, issued - NS); e < issued; ++e) mbar_wait_bounded(&bars->full[e % NS], (e / NS) & 1, a.err, 1u << 22);
        }
      }
    } else if (warp == 4 * NQ + 1) {
      // ------------------------------------------------------------------ MMA
      if (nt > 0) {
        const bool elected = elect_one();
        constexpr uint32_t idesc_s = umma_idesc_bf16(kRows, kKeys);
        constexpr uint32_t idesc_o = umma_idesc_bf16(kRows, Dh) | (1u << 16);  // B (V) is MN-major
        auto scores = [&](int w, int t, int buf, bool last) {  // S[buf] = Q_w K(t)^T
#pragma unroll
          for (int h = 0; h < E; ++h) {
            const int e = pos_k(t) * E + h, st = e % NS;
            bar_wait(&bars->dead, &bars->full[st], (e / NS) & 1, a.err);
            tc_fence_after();
            if (elected) {
              const uint64_t qd = desc_sw128(smem_u32(s_q + w * Cfg::q_bytes) + h * (CB / E) * kRows * 128, 16, 1024);
              const uint64_t kd = desc_sw128(smem_u32(s_ring + st * Cfg::entry), 16, 1024);
#pragma unroll
              for (int k = 0; k < Dh / E / 16; ++k) {
                const uint32_t off = ((k >> 2) * kRows * 128 + (k & 3) * 32) >> 4;
                umma_bf16(tmem + 256 + buf * kKeys, qd + off, kd + off, idesc_s, (h | k) != 0);
              }
              if (last) umma_commit(&bars->empty[st]);
            }
            __syncwarp();
          }
          if (elected) umma_commit(&bars->s_full[buf]);
          __syncwarp();
        };
        auto values = [&](int w, int t, int buf, int parity, bool first, bool last) {  // O_w += P[buf] V(t)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // halves of 64 keys, as the softmax hands them over
            constexpr int rows = kKeys / E;
            const int e = pos_v(t) * E + (E == 2 ? hf : 0), st = e % NS;
            if (E == 2 || hf == 0) {
              bar_wait(&bars->dead, &bars->full[st], (e / NS) & 1, a.err);
              const int live = len - tile_key(t) - (E == 2 ? hf * rows : 0);  // rows of the entry that hold a key
              if (first && live < rows) {  // the sequence ends here: what lies behind may be anything, P = 0 must stay 0
                uint8_t* v = s_ring + st * Cfg::entry;
                for (int i = lane; i < CB * rows * 8; i += 32) {
                  const int r = (i >> 3) % rows;
                  if (r >= live) *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
              }
            }
            bar_wait(&bars->dead, &bars->p_full[buf][hf], parity, a.err);
            tc_fence_after();
            if (elected) {
              const uint64_t vd = desc_sw128(smem_u32(s_ring + st * Cfg::entry) + (E == 1 ? hf * 64 * 128 : 0), rows * 128, 1024);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16_ts(tmem + w * Dh, tmem + 256 + buf * kKeys + hf * 32 + k * 8, vd + k * (2048 >> 4), idesc_o,
                             t > 0 || (hf | k) != 0);
              if (last && (E == 2 || hf == 1)) umma_commit(&bars->empty[st]);
            }
            __syncwarp();
          }
          if (elected) umma_commit(t + 1 < nt ? &bars->pv[w] : &bars->done[w]);
          __syncwarp();
        };
        bar_wait(&bars->dead, &bars->q_full, 0, a.err);
        if (NQ == 1) {
          scores(0, 0, 0, true);
          for (int t = 0; t < nt; ++t) {
            if (t + 1 < nt) scores(0, t + 1, (t + 1) & 1, true);
            values(0, t, t & 1, (t >> 1) & 1, true, true);
          }
        } else {
          for (int w = 0; w < chains; ++w) scores(w, 0, w, w == chains - 1);
          for (int t = 0; t < nt; ++t)
            for (int w = 0; w < chains; ++w) {
              values(w, t, w, t & 1, w == 0, w == chains - 1);
              if (t + 1 < nt) scores(w, t + 1, w, w == chains - 1);
            }
        }
        for (int w = 0; w < chains; ++w) mbar_wait_bounded(&bars->done[w], 0, a.err, 1u << 22);
        __syncwarp();
      }
    } else if (warp / 4 < chains) {
      // ------------------------------------------------------------------ softmax: thread = row
      const int w = warp >> 2, r = tid & 127;
      const int i_tok = tok0 + w * a.tpt + r / a.G;  // token of the chunk
      const bool valid = r < a.G * a.tpt && i_tok < n;
      const int h = kh * a.G + r % a.G, p = len - n + i_tok;
      const int pw0 = len - n + tok0 + w * a.tpt, pw1 = min(len - 1, pw0 + a.tpt - 1);  // the row tile's positions
      const uint32_t lane_base = uint32_t(warp & 3) << 21;  // TMEM lane 32 (warp % 4) in bits 16..
      const uint32_t t_o = tmem + lane_base + w * Dh;
      float m = -INFINITY, l = 0.0f;  // m: maximum in use, in units of scale2
      for (int t = 0; t < nt; ++t) {
        const int buf = NQ == 1 ? t & 1 : w, j0 = tile_key(t);
        const uint32_t t_s = tmem + lane_base + 256 + buf * kKeys;
        bar_wait(&bars->dead, &bars->s_full[buf], NQ == 1 ? (t >> 1) & 1 : t & 1, a.err);
        tc_fence_after();
        float s[kKeys];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(t_s + 32 * i, s + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_ready(s + 32 * i);
        if (j0 + kKeys - 1 > pw0 || (a.vis.window != 0 && j0 < a.vis.first(pw1))) {
          const int hi = p - j0, lw = a.vis.first(p) - j0, sk = a.vis.sinks - j0;
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (i > hi || (i < lw && i >= sk)) s[i] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < kKeys - 4; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
        mx[0] = max3(mx[0], s[kKeys - 4], s[kKeys - 3]);
        mx[1] = max3(mx[1], s[kKeys - 2], s[kKeys - 1]);
        const float top = __fmul_rn(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), a.scale2);
        if (t == 0) {
          m = top;
        } else if (__any_sync(0xFFFFFFFFu, top > m + kSlack)) {
          // O is complete once the products up to tile t - 1 are (S of tile t implies those up to t - 2)
          const float mn = top > m + kSlack ? top : m;
          const float alpha = mn == -INFINITY ? 1.0f : ex2(__fsub_rn(m, mn));
          m = mn;
          l = __fmul_rn(l, alpha);
          bar_wait(&bars->dead, &bars->pv[w], (t - 1) & 1, a.err);
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; d < Dh; d += 32) {
            float o[32];
            tmem_ld32_nowait(t_o + d, o);
            tmem_ld32_ready(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __fmul_rn(o[i], alpha);
            tmem_st16(t_o + d, reinterpret_cast<uint32_t*>(o));
            tmem_st16(t_o + d + 16, reinterpret_cast<uint32_t*>(o) + 16);
          }
        }
        const float neg = m == -INFINITY ? 0.0f : -m;  // nothing seen yet: every weight is 0
        const uint64_t scale2 = f2_pack(a.scale2, a.scale2), neg2 = f2_pack(neg, neg);
        uint64_t sum[2] = {0, 0};
        // in halves of 64 keys, each handed over as soon as it is stored
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t pk[kKeys / 4];
#pragma unroll
          for (int i = 0; i < kKeys / 4; ++i) {
            const uint64_t v = f2_fma(f2_pack(s[hf * 64 + 2 * i], s[hf * 64 + 2 * i + 1]), scale2, neg2);
            float x, y;
            if ((Cfg::poly >> (i & 7)) & 1) {
              ex2_poly(v, x, y);
            } else {
              f2_unpack(v, x, y);
              x = ex2(x);
              y = ex2(y);
            }
            sum[i & 1] = f2_add(sum[i & 1], f2_pack(x, y));
            // bf16 weights: relative error 2^-9 each, of the size of the output's own rounding; l keeps fp32
            pk[i] = pack_bf16(x, y);
          }
          tmem_st16(t_s + 32 * hf, pk);
          tmem_st16(t_s + 32 * hf + 16, pk + 16);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&bars->p_full[buf][hf]);
        }
        {
          float x, y;
          f2_unpack(f2_add(sum[0], sum[1]), x, y);
          l = __fadd_rn(l, __fadd_rn(x, y));
        }
      }
      if (nt > 0) {
        bar_wait(&bars->dead, &bars->done[w], 0, a.err);
        tc_fence_after();
      }
      // O / l, gate, store; a row with an infinity or NaN is settled by the definition afterwards
      const long long row = c0 + i_tok;
      const long long orow = (row * a.nq + h) * Dh;
      const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      float* part = a.ws_o + (long long)split * a.T * a.nq * Dh + orow;
      bool odd = false;
#pragma unroll 1
      for (int d = 0; d < Dh; d += 32) {
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        if (nt > 0) {
          tmem_ld32_nowait(t_o + d, o);
          tmem_ld32_ready(o);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) odd |= !isfinite(o[i]);
        if (valid && a.splits > 1) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(part + d + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else if (valid) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __fmul_rn(o[i], inv);
          if (a.gate) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 g4 = *reinterpret_cast<const uint4*>(a.gate + row * a.gate_ld + h * a.gate_hs + d + 8 * i);
              const uint32_t u[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                o[8 * i + 2 * x] = __fdividef(o[8 * i + 2 * x], 1.0f + ex2(-kLog2e * bflo(u[x])));
                o[8 * i + 2 * x + 1] = __fdividef(o[8 * i + 2 * x + 1], 1.0f + ex2(-kLog2e * bfhi(u[x])));
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(a.out + orow + d + 8 * i) =
                make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                           pack_bf16(o[8 * i + 4], o[8 * i + 5]), pack_bf16(o[8 * i + 6], o[8 * i + 7]));
        }
        __syncwarp();
      }
      if (valid && a.splits > 1) a.ws_ml[((long long)split * a.T + row) * a.nq + h] = make_float2(m, l);
      unsigned todo = __ballot_sync(0xFFFFFFFFu, odd && valid);
      while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        const int rr = (tid & 127 & ~31) + src, ti = tok0 + w * a.tpt + rr / a.G, hh = kh * a.G + rr % a.G;
        const long long tr = c0 + ti;
        float mm = -INFINITY, ll = 0.0f, oo[Dh / 32] = {};
        for (int t = 0; t < nt; ++t)
          attend_row_strict<Dh>(c, a.q + tr * a.q_ld + (long long)hh * Dh, b, kh, len - n + ti, tile_key(t),
                                tile_key(t) + kKeys, a.vis, a.scale2, a.err, mm, ll, oo);
        __syncwarp();
        for (int e = 0; e < Dh / 32; ++e) {
          const int d = lane * (Dh / 32) + e;
          const long long at = (tr * a.nq + hh) * Dh + d;
          if (a.splits > 1) {
            a.ws_o[(long long)split * a.T * a.nq * Dh + at] = oo[e];
          } else {
            float y = __fdiv_rn(oo[e], ll);
            if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[tr * a.gate_ld + hh * a.gate_hs + d])));
            a.out[at] = f2bf(y);
          }
        }
        if (a.splits > 1 && lane == 0) a.ws_ml[((long long)split * a.T + tr) * a.nq + hh] = make_float2(mm, ll);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4 * NQ + 1) tmem_dealloc(tmem, 512);
}

// Joins the splits of a row: one warp per (row, head), splits in order.  A row of no sequence is left alone.
template <int Dh>
__global__ void __launch_bounds__(256) prompt_join_kernel(PagedView c, PromptArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int N = Dh / 32;
  const int lane = threadIdx.x & 31;
  const long long rh = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (long long)a.T * a.nq;
  if (rh >= rows) return;
  const int row = int(rh / a.nq), h = int(rh - (long long)row * a.nq);
  bool mine = false;
  for (int i = 0; i < c.B; i += 32) {
    const int k = i + lane;
    mine |= k < c.B && a.cu[k] >= 0 && a.cu[k + 1] <= a.T && a.cu[k] <= row && row < a.cu[k + 1];
  }
  if (!__any_sync(0xFFFFFFFFu, mine)) return;
  float M = -INFINITY, l = 0.0f, o[N] = {};
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.ws_ml[s * rows + rh].x);
  const float safe = M == -INFINITY ? 0.0f : M;
  for (int s = 0; s < a.splits; ++s) {
    const float2 v = a.ws_ml[s * rows + rh];
    const float f = ex2(__fsub_rn(v.x, safe));
    l = __fmaf_rn(f, v.y, l);
    if (f == 0.0f) continue;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = __fmaf_rn(f, a.ws_o[(s * rows + rh) * Dh + lane + 32 * e], o[e]);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int d = lane + 32 * e;
    float y = l == 0.0f ? 0.0f : __fdiv_rn(o[e], l);
    if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[row * a.gate_ld + h * a.gate_hs + d])));
    a.out[rh * Dh + d] = f2bf(y);
  }
}

// ----------------------------------------------------------------------------- host
// CTAs that a call needs at most (the sequences' row counts are only known on the device).
static long long prompt_items(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  const int NQ = c->Dh == 256 ? 1 : 2, TT = NQ * (kRows / (a->n_q / c->n_kv));
  return ((long long)a->T / TT + std::min(a->T, c->B)) * c->n_kv;
}

// With fewer CTAs than SMs the key tiles of each are split, down to two tiles a split.
static int prompt_splits(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  const long long items = prompt_items(a, c), sms = sm_count();
  long long tiles = ((long long)c->table_w * c->page + kKeys - 1) / kKeys;
  if (a->window > 0) tiles = std::min(tiles, ((long long)a->window + kRows) / kKeys + 2 + a->sinks / kKeys);
  return int(std::max<long long>(1, std::min({sms / items, tiles / 2, 32ll})));
}

template <int Dh>
static int launch_prompt(const qmtp_paged_args* args, const PagedView& v, const PromptArgs& a, long long items,
                         cudaStream_t st) {
  using Cfg = PromptCfg<Dh>;
  static DeviceOnce ready;
  if (!ready([] {
        return cudaFuncSetAttribute(paged_prompt_kernel<Dh>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem);
      }))
    return QMTP_ERR_CUDA;
  CUtensorMap tq, tk, tv;
  const cuuint64_t qd[3] = {Dh, cuuint64_t(a.nq), cuuint64_t(a.T)}, qs[2] = {Dh * 2, cuuint64_t(a.q_ld) * 2};
  const cuuint32_t qb[3] = {64, cuuint32_t(a.G), cuuint32_t(a.tpt)};
  const cuuint64_t kd[2] = {Dh, cuuint64_t((v.pages * v.nkv) << v.page_log)}, ks[1] = {Dh * 2};
  const cuuint32_t kb[2] = {64, cuuint32_t(std::min(1 << v.page_log, kKeys / Cfg::E))};
  if (!encode_pages(&tq, a.q, 3, qd, qs, qb) || !encode_pages(&tk, v.k, 2, kd, ks, kb) || !encode_pages(&tv, v.v, 2, kd, ks, kb))
    return QMTP_ERR_CUDA;
  launch_kernel(paged_prompt_kernel<Dh>, dim3(unsigned(items), unsigned(a.splits)), dim3(Cfg::threads), Cfg::smem, st, tq, tk,
                tv, v, a);
  if (a.splits > 1)
    launch_kernel(prompt_join_kernel<Dh>, dim3(unsigned(((long long)a.T * a.nq + 7) / 8)), dim3(256), 0, st, v, a);
  return cudaGetLastError() == cudaSuccess ? QMTP_OK : QMTP_ERR_CUDA;
}

}  // namespace qmtp

using namespace qmtp;

static size_t prompt_o_bytes(const qmtp_paged_args* a, const qmtp_paged_cache* c, int splits) {
  return (size_t(splits) * a->T * a->n_q * c->Dh * sizeof(float) + 255) & ~size_t(255);
}

extern "C" size_t qmtp_paged_prompt_workspace(const qmtp_paged_args* args, const qmtp_paged_cache* cache) {
  PagedView v;
  if (paged_view(cache, &v) || paged_check_args(args, cache)) return 0;
  const int splits = prompt_splits(args, cache);
  if (splits == 1) return 0;
  return prompt_o_bytes(args, cache, splits) + size_t(splits) * args->T * args->n_q * sizeof(float2);
}

extern "C" int qmtp_paged_prompt(const qmtp_paged_args* args, const int* cu, const qmtp_paged_cache* cache,
                                 void* workspace, size_t ws_bytes, void* stream) {
  PagedView v;
  if (const int rc = paged_view(cache, &v)) return rc;
  if (const int rc = paged_check_args(args, cache)) return rc;
  if (!cu) return QMTP_ERR_ARG;
  const size_t need = qmtp_paged_prompt_workspace(args, cache);
  if (need && !workspace) return QMTP_ERR_ARG;
  if (ws_bytes < need) return QMTP_ERR_SHAPE;
  if (need && !aligned16(workspace)) return QMTP_ERR_ALIGN;
  const long long items = prompt_items(args, cache);
  if (items >= (1ll << 31) || (long long)args->T * args->n_q >= (1ll << 31)) return QMTP_ERR_SHAPE;
  unsigned* err = device_error_ptr();
  if (!err) return QMTP_ERR_CUDA;
  PromptArgs a{};
  a.cu = cu;
  a.q = static_cast<const uint16_t*>(args->q);
  a.gate = static_cast<const uint16_t*>(args->gate);
  a.out = static_cast<uint16_t*>(args->out);
  a.q_ld = args->q_ld ? args->q_ld : (long long)args->n_q * cache->Dh;
  a.gate_ld = args->gate_ld;
  a.gate_hs = args->gate_hs;
  a.T = args->T;
  a.nq = args->n_q;
  a.G = args->n_q / v.nkv;
  a.tpt = kRows / a.G;
  a.splits = prompt_splits(args, cache);
  a.scale2 = args->scale * kLog2e;
  a.vis = Visible{args->window, args->sinks};
  a.err = err;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + prompt_o_bytes(args, cache, a.splits));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->Dh == 64 ? launch_prompt<64>(args, v, a, items, st)
                         : cache->Dh == 128 ? launch_prompt<128>(args, v, a, items, st)
                                            : launch_prompt<256>(args, v, a, items, st);
}
