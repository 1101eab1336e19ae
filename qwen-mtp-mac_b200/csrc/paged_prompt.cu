// Prompt attention over the paged cache on the tensor cores (tcgen05), for a ragged batch of chunks.
//
// Work comes in items: two tiles of 128 query rows (128 / G tokens x the G query heads of a key head, which all read
// the same keys) and the key tiles (128 keys) that they see, walked with the running maximum m and sum l of the softmax.
// Per score tile: S = Q K^T into TMEM; the row tile's 128 threads, one row each, turn S into weights
// P = 2^(S scale2 - m) in place (bf16); O += P V with P from TMEM.  O stays in TMEM and is rescaled only when a
// row's maximum has grown by more than 2^kSlack since the last rescale, which leaves P <= 2^kSlack; the final division
// by l takes it out again.
//   warps 0 .. 4 NQ - 1   softmax, and at the end O / l, the gate and the store
//   warp 4 NQ             which item is next; TMA: pages into a ring of tiles (128-byte swizzle)
//   warps 4 NQ + 1 ..     MMA issue, by a thread for each row tile
// Each row tile has two score tiles in TMEM: the scores of the next keys run under this one's softmax.  TMEM: O in
// columns [0, 256), S in [256, 512).
//
// Dh 256: a pair of CTAs, a row tile each, 128 keys a score tile.  The tensor core takes 2048 cycles a key tile, the
// softmax 1850; 128 rows against 128 KB of keys and values would need 64 bytes a cycle of every SM, what L2 has.  So the
// pair shares each tile (cta_group::2: half of K's keys and of V's dims in each CTA), half the traffic and twice the ring.
// 16384 tokens, 16 / 4 heads of 256, causal: 1361 us, 1.62 PFLOP/s, 2166 cycles a key tile; by single CTAs 1600 us.
// Dh 128, 64: one CTA, both row tiles, 64 keys a score tile.  Here the exponentials (16 a cycle and SM) take as long as
// the products, and two warps a scheduler do not hide all of each other's latencies: 6000 tokens, 32 / 8 heads of 128:
// 283 us, 1.04 PFLOP/s (by turns that pass behind the stores 302).
#include <algorithm>

#include "paged.cuh"
#include "prompt_items.cuh"

namespace qmtp {

constexpr int kRows = 128;  // query rows of a tile
constexpr int kKeys = 128;  // keys of a tile
constexpr float kSlack = 8.0f;

template <int Dh>
struct PromptCfg {
  static constexpr bool PAIR = Dh == 256;                    // a pair of CTAs works on an item
  static constexpr int NQ = PAIR ? 1 : 2;                    // row tiles per CTA
  static constexpr int entry = kKeys * Dh * 2 * NQ / 2;      // bytes of a ring entry: a K or V tile, or the CTA's half
  static constexpr int box = kKeys * NQ / 2;                 // most rows of a copy
  static constexpr int SUB = kKeys / NQ;                     // keys of a score tile (two per row tile in TMEM)
  static constexpr int stages = Dh == 64 ? 8 : 5;
  static constexpr int threads = NQ * 128 + 32 + NQ * 32;
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
  int takes_over;             // more blocks than SMs
  float scale2;
  Visible vis;
  unsigned* err;
};

// One unit of work: a row tile (pair) of a sequence with one key head, and its share of the key tiles.
struct PromptItem {
  int b, kh, split, tok0, n, c0, len;  // b < 0: no more work
};

// PAIR: full, p_full, q_full and item_empty are used in the first CTA, where the MMAs are issued, by both CTAs' warps; the
// others tell each CTA of what happened.
struct PromptBars {
  uint64_t full[8], empty[8], q_full, q_empty, s_full[2][2], p_full[2][2][2];  // [row tile][score tile][64 keys]
  uint64_t pv[2];    // a phase per score tile but an item's last: O holds the products up to it
  uint64_t done[2];  // an item's last product
  uint64_t item_full[2], item_empty[2], next_full;
  uint64_t tail;     // PAIR: this CTA's half of a V tile in which the sequence ends
  // Two row tiles: the warps of both that share a scheduler take turns at the exponentials.  Side by side they fall into
  // step, share the exponential unit, and then leave it idle together while they wait and search maxima.
  uint64_t turn[2][4];
  alignas(16) uint4 next[1];
  PromptItem item[2];
  uint32_t tmem;
  WaitState wait;
};

// What an item's key tiles are, from its place.
struct PromptTiles {
  int p_first, p_last, chains, lo, lo_tile, sink_tiles, begin, nt, subs;
  // SUB: keys of a score tile; subs: score tiles, without one that lies wholly behind the last row
  __device__ __forceinline__ PromptTiles(const PromptItem& x, const PromptArgs& a, int NQ) {
    const int SUB = kKeys / NQ;
    p_first = x.len - x.n + x.tok0;
    p_last = x.len - x.n + min(x.n, x.tok0 + 2 * a.tpt) - 1;
    chains = NQ == 1 || x.tok0 + a.tpt >= x.n ? 1 : 2;  // row tiles that hold a token
    // key tiles: [0, sink_tiles), then [lo / 128, p_last / 128]
    lo = a.vis.first(max(p_first, 0));
    lo_tile = lo / kKeys;
    sink_tiles = a.vis.sinks > 0 && lo > 0 ? min((min(a.vis.sinks, lo) + kKeys - 1) / kKeys, lo_tile) : 0;
    const int all = p_last < 0 ? 0 : sink_tiles + p_last / kKeys + 1 - lo_tile;
    begin = int((long long)all * x.split / a.splits);
    nt = int((long long)all * (x.split + 1) / a.splits) - begin;
    subs = nt * NQ;
    if (nt > 0 && key(nt - 1) + kKeys - SUB > p_last) --subs;
  }
  __device__ __forceinline__ int key(int t) const {  // first key of the t-th tile
    t += begin;
    return (t < sink_tiles ? t : lo_tile + t - sink_tiles) * kKeys;
  }
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
// Asks for a block of this grid that has not started: it will not start, and this block does its work.  The answer
// (16 bytes) counts on `bar`.
__device__ __forceinline__ void next_block_request(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// The block's index in x, or -1: every block has started.
__device__ __forceinline__ int next_block(const void* answer) {
  uint32_t got, x = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n\t}"
      : "=r"(got), "+r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  fence_proxy_async();
  return got ? int(x) : -1;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max32(const float* s) {
  float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int i = 4; i < 28; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
  mx[0] = max3(mx[0], s[28], s[29]);
  mx[1] = max3(mx[1], s[30], s[31]);
  return fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
}
// Bits [0, n) of a word, for any n.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }
// -inf for the scores of 32 keys that the row does not see: beyond hi, or before lw and not below sk.
__device__ __forceinline__ void mask32(float* s, int hi, int lw, int sk) {
  const uint32_t keep = below(hi + 1) & (~below(lw) | below(sk));
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(keep >> i & 1)) s[i] = -INFINITY;
}
// 1 / (1 + e^-x) with the hardware's exponential and reciprocal (each within 2^-22)
__device__ __forceinline__ float sigmoid_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__fadd_rn(1.0f, ex2(__fmul_rn(-kLog2e, x)))));
  return y;
}
// Among four neighbouring lanes: lane q's v[j] becomes lane j's v[q].
__device__ __forceinline__ void transpose4(uint4 (&v)[4], int lane) {
#pragma unroll
  for (int s = 1; s <= 2; s <<= 1) {
    const bool up = (lane & s) != 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = s == 1 ? 2 * k : k, j = i + s;
      const uint4 give = up ? v[i] : v[j];
      const uint4 got = make_uint4(__shfl_xor_sync(0xFFFFFFFFu, give.x, s), __shfl_xor_sync(0xFFFFFFFFu, give.y, s),
                                   __shfl_xor_sync(0xFFFFFFFFu, give.z, s), __shfl_xor_sync(0xFFFFFFFFu, give.w, s));
      if (up) v[i] = got; else v[j] = got;
    }
  }
}
// ---- a pair of CTAs (cta_group::2): the MMAs of both are issued by the first; each holds its 128 rows of Q, S, P and O,
// and half of every K tile (64 keys) and V tile (128 dims), which the tensor cores of both read.
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
__device__ __forceinline__ uint32_t in_cta(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same without the release of this thread's memory operations (a release at cluster scope takes about 1000 cycles
// here): for tensor memory, whose order the tcgen05 fences on both sides give.
__device__ __forceinline__ void arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// warp_wait / bar_wait for what another CTA of the cluster released.
__device__ __forceinline__ bool bar_wait_cluster(WaitState* w, uint64_t* bar, uint32_t parity, unsigned* err) {
  const bool ok = bar_wait(w, bar, parity, err);
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
  return ok;
}
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int x, int y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (!PAIR) return umma_bf16(d, a, b, idesc, accumulate);
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (!PAIR) return umma_bf16_ts(d, a, b, idesc, accumulate);
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier, PAIR: in both CTAs, when the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if (!PAIR) return umma_commit(bar);
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x != 0;
}
// A sign of life to the warps that wait in this CTA and, PAIR, in the other.
template <bool PAIR>
__device__ __forceinline__ void sign_of_life_all(WaitState* w) {
  if (!PAIR) return sign_of_life(w);
  if ((threadIdx.x & 31) < 2)
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], 1;" ::"r"(in_cta(&w->alive, threadIdx.x & 31)) : "memory");
}

// Settles the rows `todo` of a softmax warp (bit = lane = row) whose O holds infinities or NaN: from values that the row
// sees, as 0 * inf from values in its tiles that it does not see, or from a sum beyond fp32.  What is finite in O is right.
// Where the row sees an infinity or NaN in a dim, that is the dim's result: found by one pass over the values that the
// warp's rows see, lane l looking after dims [l Dh / 32, (l + 1) Dh / 32) of all rows, which ends once every such dim of O
// is NaN.  Rows with a dim that no seen value explains are computed again by the definition, reading seen keys only: few,
// next to a value that is not finite and not theirs.  16384 tokens, 8 / 2 heads of 256 (0.67 ms): an infinity near the start
// 15 ms, every value NaN 1.2, a last token of NaN 180 (127 tokens by the definition).
template <int Dh>
__device__ __noinline__ void settle_rows(const PagedView c, const PromptArgs a, const PromptItem x, WaitState* wait,
                                         int tile0, uint32_t t_o, unsigned todo) {
  constexpr int N = Dh / 32, AHEAD = 8;
  constexpr bool PAIR = PromptCfg<Dh>::PAIR;
  const int lane = threadIdx.x & 31, row0 = threadIdx.x & 96;
  const PromptTiles ts(x, a, PromptCfg<Dh>::NQ);
  const bool mine = todo >> lane & 1;
  const int p = x.len - x.n + tile0 + (row0 + lane) / a.G;
  // per dim of this lane, a bit for each row: not finite in O; NaN, inf, -inf among the values seen
  unsigned odd[N], nans[N], pos[N], neg[N];
#pragma unroll
  for (int e = 0; e < N; ++e) odd[e] = nans[e] = pos[e] = neg[e] = 0;
#pragma unroll 1
  for (int d = 0; d < Dh; d += 32) {
    float o[32];
    tmem_ld32_nowait(t_o + d, o);
    tmem_ld32_ready(o);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const unsigned rows = __ballot_sync(0xFFFFFFFFu, !isfinite(o[i])) & todo;
      if (lane == (d + i) / N) odd[i % N] = rows;
    }
  }
#pragma unroll 1
  for (int t = 0; t < ts.nt; ++t) {
    const int end = min(ts.key(t) + kKeys, ts.p_last + 1);
#pragma unroll 1
    for (int j = ts.key(t); j < end; j += AHEAD) {
      unsigned seen_by[AHEAD], need = 0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        seen_by[i] = __ballot_sync(0xFFFFFFFFu, mine && j + i < end && a.vis(p, j + i));
        need |= unsigned(seen_by[i] != 0) << i;
      }
      if (need == 0) continue;
      const long long row = lane < AHEAD && (need >> lane & 1) ? cache_row(c, x.b, x.kh, j + lane, a.err) : -1;
      uint32_t v[AHEAD][N / 2];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const long long r = __shfl_sync(0xFFFFFFFFu, row, i);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) v[i][e] = 0;
        if (r >= 0) load_dims<N>(v[i], c.v + r * Dh + lane * N);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t bits = e & 1 ? v[i][e / 2] >> 16 : v[i][e / 2] & 0xFFFFu;
          if ((bits & 0x7F80u) != 0x7F80u) continue;
          if (bits & 0x7Fu)
            nans[e] |= seen_by[i];
          else if (bits & 0x8000u)
            neg[e] |= seen_by[i];
          else
            pos[e] |= seen_by[i];
        }
    }
    sign_of_life_all<PAIR>(wait);
    unsigned open = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) open |= odd[e] & ~(nans[e] | (pos[e] & neg[e]));
    if (!__any_sync(0xFFFFFFFFu, open != 0)) break;
  }
  unsigned again = 0;  // rows to compute by the definition
#pragma unroll
  for (int e = 0; e < N; ++e) again |= odd[e] & ~(nans[e] | pos[e] | neg[e]);
  again = __reduce_or_sync(0xFFFFFFFFu, again);
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const int ti = tile0 + (row0 + src) / a.G, h = x.kh * a.G + (row0 + src) % a.G, pr = x.len - x.n + ti;
    const long long tr = x.c0 + ti, orow = (tr * a.nq + h) * Dh;
    const bool redo = again >> src & 1;
    float m = -INFINITY, l = 0.0f, o[N] = {};
    if (redo)
      for (int t = 0; t < ts.nt; ++t) {
        attend_row_strict<Dh>(c, a.q + tr * a.q_ld + (long long)h * Dh, x.b, x.kh, pr, ts.key(t), ts.key(t) + kKeys, a.vis,
                              a.scale2, a.err, m, l, o);
        sign_of_life_all<PAIR>(wait);
      }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool up = pos[e] >> src & 1, down = neg[e] >> src & 1, known = up || down || (nans[e] >> src & 1);
      if (!known && !redo) continue;
      const int d = lane * N + e;
      float y = up ? INFINITY : -INFINITY;
      if ((nans[e] >> src & 1) || (up && down)) y = __int_as_float(0x7FFFFFFF);
      if (a.splits > 1) {
        a.ws_o[(long long)x.split * a.T * a.nq * Dh + orow + d] = known ? y : o[e];
        continue;
      }
      if (!known) y = pr < 0 ? 0.0f : __fdiv_rn(o[e], l);
      if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[tr * a.gate_ld + h * a.gate_hs + d])));
      a.out[orow + d] = f2bf(y);
    }
    if (redo && a.splits > 1 && lane == 0) a.ws_ml[((long long)x.split * a.T + tr) * a.nq + h] = make_float2(m, l);
  }
  __syncwarp();
}

template <int Dh>
__global__ void __launch_bounds__(PromptCfg<Dh>::threads, 1)
paged_prompt_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, PagedView c, PromptArgs a) {
  using Cfg = PromptCfg<Dh>;
  constexpr bool PAIR = Cfg::PAIR;
  constexpr int NQ = Cfg::NQ, NS = Cfg::stages, SUB = Cfg::SUB, CB = Dh / 64;  // CB: 64-dim column blocks
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* s_q = base;
  uint8_t* s_ring = base + NQ * Cfg::q_bytes;
  static_assert(sizeof(PromptBars) <= 512, "PromptCfg::smem");
  PromptBars* bars = reinterpret_cast<PromptBars*>(s_ring + NS * Cfg::entry);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  const int rank = PAIR ? int(cluster_rank()) : 0;

  if (warp == 4 * NQ + 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&bars->tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&bars->tmem, 512);
    }
  }
  if (warp == 4 * NQ && lane == 0) {
    prefetch_tensormap(&tq);
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
    for (int i = 0; i < NS; ++i) { mbar_init(&bars->full[i], 1); mbar_init(&bars->empty[i], NQ); }
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, NQ);
    mbar_init(&bars->next_full, 1);
    mbar_init(&bars->tail, 1);
    for (int i = 0; i < 8; ++i) mbar_init(&bars->turn[i >> 2][i & 3], 1);
    for (int i = 0; i < 2; ++i) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&bars->s_full[i][k], 1);
        mbar_init(&bars->p_full[i][k][0], PAIR ? 8 : 128);
        mbar_init(&bars->p_full[i][k][1], PAIR ? 8 : 128);
      }
      mbar_init(&bars->pv[i], 1);
      mbar_init(&bars->done[i], 1);
      mbar_init(&bars->item_full[i], 1);
      mbar_init(&bars->item_empty[i], 10);  // a pair: 4 + 1 warps each; else 8 + 2
    }
    bars->wait = WaitState{0, 0};
    fence_mbar_init();
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the barriers of both CTAs are ready
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  // ring position, within an item, of K(t), V(t): Dh 256 loads K0 K1 V0 K2 V1 ..., otherwise K0 V0 K1 V1 ...
  auto pos_k = [&](int t) { return NQ == 1 ? (t == 0 ? 0 : 2 * t - 1) : 2 * t; };
  auto pos_v = [&](int t, int nt) { return NQ == 1 ? min(2 * t + 2, 2 * nt - 1) : 2 * t + 1; };

  if (warp == 4 * NQ) {
    // -------------------------------------------------------------------- items and TMA
    const int TT = 2 * a.tpt;                                             // tokens per item
    const int box = min(1 << c.page_log, Cfg::box), parts = kKeys / box;  // rows per box, boxes down a tile
    const long long none = (c.pages * c.nkv) << c.page_log;                // past the end: reads as zeros
    ItemCursor at_seq;
    int e0 = 0, issued = 0, loads = 0, tails = 0, asked = 0;
    long long u = blockIdx.x / (PAIR ? 2 : 1);
    bool own = true;  // the block's own place, not one that it took over
    for (int i = 0;;) {
      // The next item: that of a block of the grid that has not started, taken over while this one runs.  With no more
      // blocks than SMs each finds a place of its own, and none is taken.
      if (lane == 0 && rank == 0 && a.takes_over) {
        mbar_expect_tx(&bars->next_full, 16);
        next_block_request(bars->next, &bars->next_full);
      }
      PromptItem x;
      x.b = -1;
      x.split = int(u % a.splits);
      x.kh = int(u / a.splits % c.nkv);
      const long long tile = u / a.splits / c.nkv;
      at_seq.seek(tile);
      while ((rank == 0 || own) && at_seq.seq < c.B) {
        const int k = at_seq.seq + lane;
        int n = 0, c0 = 0, len = 0;
        if (k < c.B) {
          c0 = a.cu[k];
          const int c1 = a.cu[k + 1];
          len = seq_len(c, k, a.err);
          n = c1 - c0;
          if (c0 < 0 || c1 > a.T || c1 < c0) {
            atomicOr(a.err, DEVERR_BADARG);
            n = 0;
          }
        }
        const int tiles = (n + TT - 1) / TT;
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
          if (lane >= d) incl += y;
        }
        const long long at = tile - at_seq.before - (incl - tiles);
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, at >= 0 && at < tiles);
        if (hit) {
          const int src = __ffs(hit) - 1;
          x.b = at_seq.seq + src;
          x.n = __shfl_sync(0xFFFFFFFFu, n, src);
          x.c0 = __shfl_sync(0xFFFFFFFFu, c0, src);
          x.len = __shfl_sync(0xFFFFFFFFu, len, src);
          x.tok0 = (__shfl_sync(0xFFFFFFFFu, tiles, src) - 1 - int(__shfl_sync(0xFFFFFFFFu, int(at), src))) * TT;
          break;
        }
        at_seq.pass(32, __shfl_sync(0xFFFFFFFFu, incl, 31));
      }
      auto take_over = [&] {  // the block that the request of this round has got, or -1
        int next = -1;
        if (a.takes_over && bar_wait(&bars->wait, &bars->next_full, asked & 1, a.err)) next = next_block(bars->next);
        ++asked;
        return __shfl_sync(0xFFFFFFFFu, next, 0);
      };
      auto hand_out = [&](const PromptItem& y, int at) {
        const bool ok = warp_wait(&bars->wait, &bars->item_empty[at & 1], ((at >> 1) & 1) ^ 1, a.err);
        if (lane == 0) {
          bars->item[at & 1] = y;
          mbar_arrive(&bars->item_full[at & 1]);
          if (PAIR && rank == 0 && (!own || y.b < 0)) {
            const uint32_t to = in_cta(&bars->item[at & 1], 1);
            const int v[7] = {y.b, y.kh, y.split, y.tok0, y.n, y.c0, y.len};
#pragma unroll
            for (int k = 0; k < 7; ++k) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + 4 * k), "r"(v[k]) : "memory");
            arrive_cluster(in_cta(&bars->item_full[at & 1], 1));
          }
        }
        __syncwarp();
        return ok;
      };
      if (rank == 0 && x.b < 0) {  // a place without rows (the grid has as many as there can be): on with the next
        const int next = take_over();
        if (next >= 0) {
          u = next / (PAIR ? 2 : 1);
          own = false;
          continue;
        }
        hand_out(x, i);
        break;
      }
      bool ok;
      if (rank == 0 || (own && x.b >= 0)) {
        ok = hand_out(x, i);
      } else {  // the second CTA finds the block's own item itself and is told of the others
        ok = __all_sync(0xFFFFFFFFu, bar_wait_cluster(&bars->wait, &bars->item_full[i & 1], (i >> 1) & 1, a.err));
        if (!ok) break;
        x = bars->item[i & 1];
        __syncwarp();
      }
      if (rank == 1 && lane == 0) arrive_cluster(in_first_cta(&bars->item_empty[i & 1]));
      const PromptTiles ts(x, a, NQ);
      if (ok && x.b >= 0 && ts.nt > 0) {
        // cache row of part `lane` of the tile at key j (a page that no row needs is not looked at)
        auto part_row = [&](int j) -> int {
          const int key = j + lane * box;
          if (lane >= parts || key > ts.p_last || (a.vis.window != 0 && key + box <= ts.lo && key >= a.vis.sinks))
            return int(none);
          const long long r = cache_row(c, x.b, x.kh, key, a.err);
          return int(r < 0 ? none : r);
        };
        auto load = [&](const CUtensorMap* map, int pos, bool is_v, int row, bool tail) {
          const int e = e0 + pos, st = e % NS;
          if (!warp_wait(&bars->wait, &bars->empty[st], ((e / NS) & 1) ^ 1, a.err)) return;
          // PAIR: the copies of both CTAs count on the first one's barrier; those of a V tile in which the sequence ends
          // on their own CTA's, whose softmax warps clear it and answer with their weights.  The barrier is free again
          // once the item before (number loads - 2) is done: its last product took every warp's weights.
          if (PAIR && tail && loads > 1 && !warp_wait(&bars->wait, &bars->done[0], loads & 1, a.err)) return;
          if (lane == 0) {
            if (PAIR && tail) mbar_expect_tx(&bars->tail, Cfg::entry);
            if (PAIR && tail && rank == 0) mbar_arrive(&bars->full[st]);
            if (!(PAIR && tail) && rank == 0) mbar_expect_tx(&bars->full[st], Cfg::entry * (PAIR ? 2 : 1));
          }
          __syncwarp();
          issued = e + 1;
          uint8_t* dst = s_ring + st * Cfg::entry;
          // an entry: a tile, or for a pair 64 of K's keys with all dims, all of V's keys with 128 dims
          const int ncb = PAIR && is_v ? CB / 2 : CB, np = PAIR && !is_v ? parts / 2 : parts, rows = PAIR && !is_v ? kKeys / 2 : kKeys;
          const int part = lane / ncb, cb = lane - part * ncb;
          const int r = __shfl_sync(0xFFFFFFFFu, row, (PAIR && !is_v ? rank * np : 0) + min(part, np - 1));
          if (part < np) {
            uint8_t* to = dst + cb * rows * 128 + part * box * 128;
            const int col = (PAIR && is_v ? rank * ncb + cb : cb) * 64;
            if (PAIR && !tail)
              tma_load_2d_pair(to, map, col, r, in_first_cta(&bars->full[st]), policy_evict_last());
            else
              tma_load_2d(to, map, col, r, PAIR ? &bars->tail : &bars->full[st], policy_evict_last());
          }
          if (tail) ++tails;
        };
        auto load_q = [&] {
          if (!warp_wait(&bars->wait, &bars->q_empty, (loads & 1) ^ 1, a.err)) return;
          if (lane == 0 && rank == 0) mbar_expect_tx(&bars->q_full, uint32_t(PAIR ? 2 : ts.chains) * a.G * a.tpt * Dh * 2);
          __syncwarp();
          if (lane < ts.chains * CB) {
            const int w = lane / CB, cb = lane - w * CB;
            uint8_t* to = s_q + w * Cfg::q_bytes + cb * kRows * 128;
            const int z = x.c0 + x.tok0 + (PAIR ? rank : w) * a.tpt;
            if (PAIR)
              tma_load_3d_pair(to, &tq, cb * 64, x.kh * a.G, z, in_first_cta(&bars->q_full));
            else
              tma_load_3d(to, &tq, cb * 64, x.kh * a.G, z, &bars->q_full);
          }
          ++loads;
        };
        auto ends = [&](int t) { return ts.key(t) + kKeys > x.len; };
        const bool first = loads == 0;
        if (first) load_q();  // later its place is still in use: behind the first keys
        int row = part_row(ts.key(0)), row_next = ts.nt > 1 ? part_row(ts.key(1)) : 0;
        load(&tk, pos_k(0), false, row, false);
        if (!first) load_q();
        for (int t = 0; t < ts.nt; ++t) {
          const int row_after = t + 2 < ts.nt ? part_row(ts.key(t + 2)) : 0;
          if (NQ == 2) load(&tv, pos_v(t, ts.nt), true, row, false);
          if (t + 1 < ts.nt) load(&tk, pos_k(t + 1), false, row_next, false);
          if (NQ == 1) load(&tv, pos_v(t, ts.nt), true, row, ends(t));
          row = row_next;
          row_next = row_after;
        }
        e0 += 2 * ts.nt;
      }
      ++i;
      own = false;
      if (rank == 1) {
        if (x.b < 0) break;
        continue;
      }
      const int next = take_over();
      if (!ok) break;
      if (next < 0) {
        x.b = -1;
        hand_out(x, i);
        break;
      }
      u = next / (PAIR ? 2 : 1);
    }
    if (given_up(&bars->wait)) {  // copies in flight end before the CTA does
      if (a.takes_over && asked > 0) mbar_wait_bounded(&bars->next_full, (asked - 1) & 1, a.err, 1u << 22);
      if (tails > 0) mbar_wait_bounded(&bars->tail, (tails - 1) & 1, a.err, 1u << 22);
      if (loads > 0 && rank == 0) mbar_wait_bounded(&bars->q_full, (loads - 1) & 1, a.err, 1u << 22);
      for (int e = rank ? issued : max(0, issued - NS); e < issued; ++e)
        mbar_wait_bounded(&bars->full[e % NS], (e / NS) & 1, a.err, 1u << 22);
    }
  } else if (warp > 4 * NQ) {
    // -------------------------------------------------------------------- MMA: a thread per row tile
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(PAIR ? 2 * kRows : kRows, SUB);
      constexpr uint32_t idesc_o = umma_idesc_bf16(PAIR ? 2 * kRows : kRows, Dh) | (1u << 16);  // B (V) is MN-major
      const int w = warp - 4 * NQ - 1;
      const uint32_t t_s = tmem + 256 + 2 * w * SUB, t_o = tmem + w * Dh;
      const uint64_t qd = desc_sw128(smem_u32(s_q + w * Cfg::q_bytes), 16, 1024);
      int e0 = 0, work = 0, g = 0, finished = 0;  // g: score tiles so far
      for (int items = 0;; ++items) {
        if (!bar_wait(&bars->wait, &bars->item_full[items & 1], (items >> 1) & 1, a.err)) break;
        const PromptItem x = bars->item[items & 1];
        mbar_arrive(&bars->item_empty[items & 1]);
        if (x.b < 0) break;
        const PromptTiles ts(x, a, NQ);
        const int nt = ts.nt, subs = ts.subs;
        if (nt > 0 && w < ts.chains) {
          auto used = [&](uint64_t* bar) { mma_commit<PAIR>(bar); };  // an entry is free when both row tiles have used it
          auto scores = [&](int j) {  // S = Q K^T of score tile j
            const int buf = (g + j) & 1, t = j / NQ, r0 = (j - t * NQ) * SUB, e = e0 + pos_k(t), st = e % NS;
            if (r0 == 0) bar_wait(&bars->wait, &bars->full[st], (e / NS) & 1, a.err);
            tc_fence_after();
            const uint64_t kd = desc_sw128(smem_u32(s_ring + st * Cfg::entry) + r0 * 128, 16, 1024);
#pragma unroll
            for (int k = 0; k < Dh / 16; ++k)
              mma_ss<PAIR>(t_s + buf * SUB, qd + (((k >> 2) * kRows * 128 + (k & 3) * 32) >> 4),
                           kd + (((k >> 2) * (PAIR ? kKeys / 2 : kKeys) * 128 + (k & 3) * 32) >> 4), idesc_s, k != 0);
            mma_commit<PAIR>(&bars->s_full[w][buf]);
            if (j % NQ == NQ - 1 || j + 1 == subs) used(&bars->empty[st]);
            if (j + 1 == subs) used(&bars->q_empty);
          };
          auto values = [&](int j) {  // O += P V of score tile j
            const int buf = (g + j) & 1, t = j / NQ, r0 = (j - t * NQ) * SUB, e = e0 + pos_v(t, nt), st = e % NS;
            if (r0 == 0) bar_wait(&bars->wait, &bars->full[st], (e / NS) & 1, a.err);
#pragma unroll
            for (int hf = 0; hf < SUB / 64; ++hf) {  // 64 keys, as the softmax hands them over
              bar_wait(&bars->wait, &bars->p_full[w][buf][hf], ((g + j) >> 1) & 1, a.err);
              tc_fence_after();
              const uint64_t vd = desc_sw128(smem_u32(s_ring + st * Cfg::entry) + (r0 + hf * 64) * 128, kKeys * 128, 1024);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_ts<PAIR>(t_o, t_s + buf * SUB + hf * 32 + k * 8, vd + k * (2048 >> 4), idesc_o, j > 0 || (hf | k) != 0);
            }
            mma_commit<PAIR>(j + 1 < subs ? &bars->pv[w] : &bars->done[w]);
            if (j % NQ == NQ - 1 || j + 1 == subs) used(&bars->empty[st]);
          };
          bar_wait(&bars->wait, &bars->q_full, work & 1, a.err);
          // S0 S1 | O0 S2 | O1 S3 ...: the next scores are always under way while the softmax works
          for (int j = 0; j < min(2, subs); ++j) scores(j);
          for (int j = 0; j < subs; ++j) {
            values(j);
            if (j + 2 < subs) scores(j + 2);
          }
          g += subs;
          ++finished;
        } else if (nt > 0) {
          // A row tile without tokens: its thread follows the item's barriers all the same.  A wait by parity is only right
          // for the phase after the last one that its thread has seen: behind a skipped item it could pass while the item's own
          // copies were under way, and the next one's products read tiles that were not there.
          bar_wait(&bars->wait, &bars->q_full, work & 1, a.err);
          mbar_arrive(&bars->q_empty);
          for (int e = e0; e < e0 + 2 * nt; ++e) {
            bar_wait(&bars->wait, &bars->full[e % NS], (e / NS) & 1, a.err);
            mbar_arrive(&bars->empty[e % NS]);
          }
        }
        if (nt > 0) ++work;
        e0 += 2 * nt;
      }
      // every product is over before the tensor memory is given back
      if (finished > 0) mbar_wait_bounded(&bars->done[w], (finished - 1) & 1, a.err, 1u << 22);
    }
    __syncwarp();
  } else if (warp < 4 * NQ) {
    // -------------------------------------------------------------------- softmax: thread = row
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lane_base = uint32_t(warp & 3) << 21;  // TMEM lane 32 (warp % 4) in bits 16..
    const uint32_t t_o = tmem + lane_base + w * Dh;
    int g = 0, pvs = 0, finished = 0;  // score tiles, phases of pv and of done so far
    int e0 = 0, tails = 0;             // ring entries of the items so far, V tiles cleared
    int turns = 0;
    for (int items = 0;; ++items) {
      if (!__all_sync(0xFFFFFFFFu, PAIR ? bar_wait_cluster(&bars->wait, &bars->item_full[items & 1], (items >> 1) & 1, a.err)
                                        : bar_wait(&bars->wait, &bars->item_full[items & 1], (items >> 1) & 1, a.err)))
        break;
      const PromptItem x = bars->item[items & 1];
      __syncwarp();
      if (lane == 0) {
        if (PAIR)
          arrive_cluster(in_first_cta(&bars->item_empty[items & 1]));
        else
          mbar_arrive(&bars->item_empty[items & 1]);
      }
      if (x.b < 0) break;
      const PromptTiles ts(x, a, NQ);
      const int e_item = e0;
      e0 += 2 * ts.nt;
      if (w >= ts.chains) continue;
      const int tile0 = x.tok0 + (PAIR ? rank : w) * a.tpt;    // the row tile's first token of the chunk
      const int nt = ts.nt, i_tok = tile0 + r / a.G;
      const bool valid = r < a.G * a.tpt && i_tok < x.n;
      const int h = x.kh * a.G + r % a.G, p = x.len - x.n + i_tok;
      const int pw0 = x.len - x.n + tile0, pw1 = min(x.len - 1, pw0 + a.tpt - 1);  // the row tile's positions
      float m = -INFINITY, l = 0.0f;  // m: maximum in use, in units of scale2
      for (int j = 0; j < ts.subs; ++j) {
        const int buf = (g + j) & 1, t = j / NQ, r0 = (j - t * NQ) * SUB, j0 = ts.key(t) + r0;
        const uint32_t t_s = tmem + lane_base + 256 + (2 * w + buf) * SUB;
        warp_wait(&bars->wait, &bars->s_full[w][buf], ((g + j) >> 1) & 1, a.err);
        tc_fence_after();
        float s[SUB];
#pragma unroll
        for (int i = 0; i < SUB; i += 32) tmem_ld32_nowait(t_s + i, s + i);
        if (j0 + SUB > x.len) {
          // The sequence ends in this tile: the values behind its end may be anything, and their weight 0 has to stay
          // 0.  They are cleared before the weights are handed over.
          const int e = e_item + pos_v(t, nt), st = e % NS;
          warp_wait(&bars->wait, PAIR ? &bars->tail : &bars->full[st], PAIR ? tails & 1 : (e / NS) & 1, a.err);
          ++tails;
          for (int i = r; i < Cfg::entry / 16 / kKeys * SUB; i += 128) {
            const int row = (i >> 3) % SUB, cb = (i >> 3) / SUB;
            if (j0 + row >= x.len)
              *reinterpret_cast<uint4*>(s_ring + st * Cfg::entry + ((cb * kKeys + r0 + row) * 8 + (i & 7)) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          if (PAIR) asm volatile("fence.acq_rel.cluster;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < SUB; i += 32) tmem_ld32_ready(s + i);
        if (j0 + SUB - 1 > pw0 || (a.vis.window != 0 && j0 < a.vis.first(pw1))) {
          const int hi = p - j0, lw = a.vis.first(p) - j0, sk = a.vis.sinks - j0;
#pragma unroll
          for (int i = 0; i < SUB; i += 32) mask32(s + i, hi - i, lw - i, sk - i);
        }
        float top = max32(s);
#pragma unroll
        for (int i = 32; i < SUB; i += 32) top = fmaxf(top, max32(s + i));
        top = __fmul_rn(top, a.scale2);
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xFFFFFFFFu, top > m + kSlack)) {
          // O is complete once the products up to tile j - 1 are (S of tile j implies those up to j - 2)
          const float mn = top > m + kSlack ? top : m;
          const float alpha = mn == -INFINITY ? 1.0f : ex2(__fsub_rn(m, mn));
          m = mn;
          l = __fmul_rn(l, alpha);
          warp_wait(&bars->wait, &bars->pv[w], (pvs + j - 1) & 1, a.err);
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
        if (NQ == 2 && ts.chains == 2) {  // the k-th time: row tile 1 behind tile 0's k-th, tile 0 behind tile 1's (k - 1)-th
          if (w == 1 || turns > 0) warp_wait(&bars->wait, &bars->turn[w][warp & 3], (turns - 1 + w) & 1, a.err);
          ++turns;
        }
#pragma unroll
        for (int c = 0; c < SUB / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x, y;
            f2_unpack(f2_fma(f2_pack(s[32 * c + 2 * i], s[32 * c + 2 * i + 1]), scale2, neg2), x, y);
            x = ex2(x);
            y = ex2(y);
            sum[i & 1] = f2_add(sum[i & 1], f2_pack(x, y));
            // bf16 weights: off by at most 2^-8 relative each, as the output's own rounding is; l keeps fp32
            pk[i] = pack_bf16(x, y);
          }
          // the turn ends with the exponentials: behind the stores the other tile would wait for them too (159 for 154 us)
          if (NQ == 2 && c == SUB / 32 - 1 && ts.chains == 2 && lane == 0) mbar_arrive(&bars->turn[w ^ 1][warp & 3]);
          tmem_st16(t_s + 16 * c, pk);
          if (c & 1) {  // 64 keys are handed over as soon as they are stored
            tmem_st_wait();
            tc_fence_before();
            if (PAIR) {
              __syncwarp();
              if (lane == 0) arrive_cluster_relaxed(in_first_cta(&bars->p_full[w][buf][c >> 1]));
            } else {
              mbar_arrive(&bars->p_full[w][buf][c >> 1]);
            }
          }
        }
        float x, y;
        f2_unpack(f2_add(sum[0], sum[1]), x, y);
        l = __fadd_rn(l, __fadd_rn(x, y));
      }
      // Four lanes share their rows' stores and gate loads: lane q of the four takes the q-th 16 bytes of 64 of each row.
      const long long row = x.c0 + i_tok;
      const bool gated = a.gate && a.splits == 1;
      long long o_off[4], g_off[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int src = (lane & ~3) + j;
        const long long rj = __shfl_sync(0xFFFFFFFFu, valid ? row : -1, src);
        const int hj = __shfl_sync(0xFFFFFFFFu, h, src);
        o_off[j] = rj < 0 ? -1 : (rj * a.nq + hj) * Dh + 8 * (lane & 3);
        g_off[j] = rj * a.gate_ld + hj * a.gate_hs + 8 * (lane & 3);
      }
      constexpr int AHEAD = 2;  // chunks of 32 dims whose gates are fetched ahead
      uint4 gates[AHEAD][4];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (gated && o_off[j] >= 0) gates[k][j] = *reinterpret_cast<const uint4*>(a.gate + g_off[j] + 32 * k);
      g += ts.subs;
      if (nt > 0) {
        pvs += ts.subs - 1;
        warp_wait(&bars->wait, &bars->done[w], finished & 1, a.err);
        ++finished;
        tc_fence_after();
      }
      // O / l, gate, store; a row with an infinity or NaN in O is settled afterwards
      const long long orow = (row * a.nq + h) * Dh;
      const float inv = p < 0 ? 0.0f : __fdiv_rn(1.0f, l);  // l = 0 at p >= 0: every score seen is -inf, 0 / 0
      float* part = a.ws_o + (long long)x.split * a.T * a.nq * Dh + orow;
      float probe[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // 0 unless O holds an infinity or NaN
#pragma unroll 2  // not more: code that runs once an item costs instruction fetches (8 chunks unrolled: +2 us)
      for (int d = 0; d < Dh; d += 32) {
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = gates[d / 32 % AHEAD][j];
          if (gated && d + 32 * AHEAD < Dh && o_off[j] >= 0)
            gates[d / 32 % AHEAD][j] = *reinterpret_cast<const uint4*>(a.gate + g_off[j] + d + 32 * AHEAD);
        }
        if (nt > 0) {
          tmem_ld32_nowait(t_o + d, o);
          tmem_ld32_ready(o);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) probe[i & 3] = __fmaf_rn(o[i], 0.0f, probe[i & 3]);
        if (a.splits > 1) {
          if (valid)
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part + d + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __fmul_rn(o[i], inv);
          if (gated) {
            transpose4(v, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[8 * i + 2 * k] = __fmul_rn(o[8 * i + 2 * k], sigmoid_fast(bflo(u[k])));
                o[8 * i + 2 * k + 1] = __fmul_rn(o[8 * i + 2 * k + 1], sigmoid_fast(bfhi(u[k])));
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                              pack_bf16(o[8 * i + 4], o[8 * i + 5]), pack_bf16(o[8 * i + 6], o[8 * i + 7]));
          transpose4(v, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (o_off[j] >= 0) *reinterpret_cast<uint4*>(a.out + o_off[j] + d) = v[j];
        }
        __syncwarp();
      }
      const bool odd = !(probe[0] + probe[1] + probe[2] + probe[3] == 0.0f);
      if (valid && a.splits > 1) a.ws_ml[((long long)x.split * a.T + row) * a.nq + h] = make_float2(m, l);
      // a sum l that is NaN makes the whole row NaN, which it is; one of 0 leaves zeros or NaN, except behind NaN in O
      const unsigned todo =
          __ballot_sync(0xFFFFFFFFu, odd && valid && l == l && (l != 0.0f || (p < 0 && a.splits == 1)));
      if (todo) settle_rows<Dh>(c, a, x, &bars->wait, tile0, t_o, todo);
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // neither CTA's memory is used by the other any more
  tc_fence_after();
  if (warp == 4 * NQ + 1) {
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else
      tmem_dealloc(tmem, 512);
  }
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
  bool mine = false, sees = false;  // the row is one of a sequence; its position is one, so it sees at least its own key
  for (int i = 0; i < c.B; i += 32) {
    const int k = i + lane;
    if (k < c.B && a.cu[k] >= 0 && a.cu[k + 1] <= a.T && a.cu[k] <= row && row < a.cu[k + 1]) {
      mine = true;
      sees = seq_len(c, k, nullptr) - a.cu[k + 1] + row >= 0;
    }
  }
  if (!__any_sync(0xFFFFFFFFu, mine)) return;
  sees = __any_sync(0xFFFFFFFFu, sees);
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
    float y = sees ? __fdiv_rn(o[e], l) : 0.0f;
    if (a.gate) y = __fmul_rn(y, sigmoid_f32(bf2f(a.gate[row * a.gate_ld + h * a.gate_hs + d])));
    a.out[rh * Dh + d] = f2bf(y);
  }
}

// ----------------------------------------------------------------------------- host
// Items of work that a call has at most (the sequences' row counts are only known on the device).
static long long prompt_items(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  const int TT = 2 * (kRows / (a->n_q / c->n_kv));
  return ((long long)a->T / TT + std::min(a->T, c->B)) * c->n_kv;
}

// With fewer items than SMs the key tiles of each are split, down to four tiles a split: two (512 tokens of 16 / 4
// heads of 256 in 128 CTAs) measured 25.1 us, whole items (64 CTAs) 18.1; 128 tokens behind 8000 want the split, 38 for 117 us.
// The host knows how many tokens the table's rows can hold, not the lengths: in a table with room to spare short prompts
// are split for nothing (those 512 tokens, in a graph: 14.4 us in a table of 512 tokens, 23.1 in one of 1024 and more).
static int prompt_splits(const qmtp_paged_args* a, const qmtp_paged_cache* c) {
  const long long items = prompt_items(a, c), sms = c->Dh == 256 ? sm_count() / 2 : sm_count();
  long long tiles = ((long long)c->table_w * c->page + kKeys - 1) / kKeys;
  if (a->window > 0) tiles = std::min(tiles, ((long long)a->window + kRows) / kKeys + 2 + a->sinks / kKeys);
  return int(std::max<long long>(1, std::min({sms / items, tiles / 4, 32ll})));
}

template <int Dh>
static int launch_prompt(const qmtp_paged_args* args, const PagedView& v, PromptArgs a, long long items,
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
  const cuuint32_t kb[2] = {64, cuuint32_t(std::min(1 << v.page_log, Cfg::box))};
  if (!encode_pages(&tq, a.q, 3, qd, qs, qb) || !encode_pages(&tk, v.k, 2, kd, ks, kb) || !encode_pages(&tv, v.v, 2, kd, ks, kb))
    return QMTP_ERR_CUDA;
  constexpr int per = Cfg::PAIR ? 2 : 1;  // CTAs of an item
  a.takes_over = items * a.splits * per > sm_count();
  launch_kernel_cluster(paged_prompt_kernel<Dh>, dim3(unsigned(items * a.splits * per)), dim3(Cfg::threads), Cfg::smem, st, per,
                        tq, tk, tv, v, a);
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
