// Attention of a drafted tree over a key/value cache (tabby_tree_attention_async).
//
//   out[b][j][h] = sum_t softmax_t(scale q.k[t]) v[t],  t < L or t = L + (j or an ancestor)
//
// The query rows of one key/value head -- slots times grouped heads, M = nodes * group of them
// -- share its keys, so a tile of 128 rows is the M of two tensor-core products, S = Q K^T and
// O += P V, over tiles of 64 keys, and the caches are read once. Between the products the
// softmax runs in one pass: a running maximum m and sum l a row,
//   P = 2^(c S - m),  l += sum P,  and where the maximum rises: O, l *= 2^(m_old - m),
// c = scale log2(e), m = c max S. The maximum is only moved when it rises by more than 8 in the
// exponent (P then stays below 2^8), so O is rarely rescaled. l sums P in fp32; for the product P
// is rounded to the inputs' type, since both operands of a 16-bit product have it and one of 32 bits
// runs at half the rate from V's tiles widened to twice their bytes. (Outputs off by 0.0021 to
// 0.0023 in bf16 and 0.00029 in fp16, relative in the norm, where the rounding of the outputs alone
// makes 0.0017 and 0.00021.)
//
//   tree_kernel      one CTA a worker. The work of a call --
//                    every (sequence, key/value head, row tile) has ceil((L + nodes) / 64) key
//                    tiles -- is laid end to end and cut into equal ranges, one a worker, from
//                    the lengths on the device: long and short sequences load the SMs evenly
//                    and a single long one is spread over all of them.
//                    warps 0-3   softmax: thread r owns row r (TMEM lane r). S by tcgen05.ld,
//                                P back to TMEM as 16-bit values over S's columns; writes Q's
//                                tile and, at a range's or item's end, the row's result.
//                    warp 4      TMA producer: 4-D loads of K and V tiles (64 keys x 64 values
//                                a box, 128-byte swizzle, zero fill past the cache) into two
//                                rings.
//                    last warps  tcgen05.mma issuers, one a row tile: S double-buffered (the next tile's S is
//                                computed while this one's softmax runs), O in TMEM.
//   tree_join_kernel joins the parts of items that were cut between workers.
//
// A bounded wait that runs out makes the CTA give up: what it had not finished becomes NaN.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "decode_internal.h"
#include "sm100.cuh"

namespace tabby {
namespace {

constexpr int kTileT = 64;        // keys a tile
constexpr int kTileM = 128;       // query rows a tile (the MMA's M, TMEM's lanes)
// Workers at most, which bounds the workspace: two an SM, one where two row tiles go together.
constexpr int max_workers(int64_t mrows) { return mrows > 128 ? 160 : 320; }
constexpr float kLazy = 8.f;      // the maximum moves when it rises by more than 2^8

// Builds that check themselves (-DTABBY_CHECKS=1) can make waits of one sequence's tiles run out
// (tabby_debug_tree): its value tiles are never loaded, or the first issuer gives up behind a
// product of it that it has just issued. Every wait is bounded, so the kernel returns all the same.
// They count the CTAs that would give their TMEM back with a product on its way.
#ifdef TABBY_CHECKS
struct TreeChecks {
  int withhold, give_up;  // sequences, -1: none
  int in_flight;
};
__device__ TreeChecks g_tree_checks = {-1, -1, 0};
#endif

// A worker for heads of up to DP values that takes NS row tiles together: they share every K
// and V tile. One row tile: two workers an SM; two: one.
template <int DP, int NS>
struct TreeCfg {
  static constexpr int kThreads = 160 * NS + 32;
  static constexpr int kBlocks = DP / 64;             // blocks of 64 values: one swizzle row
  static constexpr int kQ = kTileM * 128 * kBlocks;   // bytes of a Q tile
  static constexpr int kKv = kTileT * 128 * kBlocks;  // bytes of a K or V tile
  static constexpr int kStages = NS == 1 ? (DP == 64 ? 5 : 2) : (DP == 64 ? 8 : 5);
  static constexpr int kRings = 2 * kStages * kKv;    // K's and V's tiles
  static constexpr size_t kSmem = 1024 + NS * kQ + kRings + 1024;
  // TMEM columns: a row tile's O, then its two S tiles.
  static constexpr uint32_t kO = 0, kS = NS * DP;
  static constexpr uint32_t kTmem = NS == 1 ? 256 : 512;
  static_assert(kS + NS * 2 * kTileT <= kTmem, "TMEM columns");
};

struct TreeArgs {
  tabby_tree_attention_args u;
  int32_t group;    // heads a key/value head
  uint32_t by_group;  // ceil(2^32 / group): division by it as a product, group 2 to 256
  int32_t mrows;    // query rows of a key/value head
  int32_t mtiles;   // row tiles of a key/value head, those that go together as one
  int32_t workers;  // CTAs the key tiles are cut over
  int32_t prow;     // rows a part holds: min(mrows, 128 a row tile)
  float c;          // |scale| log2(e), 1 where scale is 0
  uint32_t q_xor;   // flips the signs of Q's values where scale is negative
  uint32_t q_and;   // 0 where scale is 0
  float *part_o;    // [2 * workers][dim / 4][prow][4]: unscaled sums
  float2 *part_ml;  // [2 * workers][prow]: m, sum
  // Items that were cut: sequence, head and row tile (head * mtiles + row tile), the first part's
  // slot, the parts (0: none). By item where there are no more of them than workers; else by the
  // worker that has the first part (no worker begins two cut items).
  int4 *cuts;
  int32_t items, by_item;
};

// y / group for a row y < 64 * group (and up to 255 more): with 2^32 / group rounded up the
// product is above y / group by less than y / 2^32, below 1 / group while y * group < 2^32.
__device__ __forceinline__ int div_group(const TreeArgs &a, int y) {
  if (a.group == 1) return y;  // 2^32 has no place in by_group
  return a.group <= 256 ? (int)__umulhi((uint32_t)y, a.by_group) : y / a.group;
}

// Key tiles of one (head, row tile) of a sequence; 0: nothing to attend to.
__device__ __forceinline__ int seq_tiles(const TreeArgs &a, int b) {
  const int L = a.u.lengths[b];
  if (L < 0 || L >= a.u.entries) return 0;
  const int n = a.u.entries - L > a.u.nodes ? L + a.u.nodes : a.u.entries;
  return (n - 1) / kTileT + 1;
}
// Sums over the sequences, 32 at a time, a lane each; all lanes call. With x < 0: the key tiles
// of the call. Else where tile x lies: its sequence, and the number of tiles before it.
__device__ __forceinline__ int scan_tiles(const TreeArgs &a, int first32, int x, int &b) {
  const int lane = threadIdx.x & 31;
  const int per = a.u.kv_heads * a.mtiles;
  int t0 = 0;
  for (int b0 = 0; b0 < a.u.batch; b0 += 32) {
    const int n = per * (b0 == 0 ? first32 : b0 + lane < a.u.batch ? seq_tiles(a, b0 + lane) : 0);
    int end = n;  // inclusive prefix sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += y;
    }
    const unsigned in = __ballot_sync(0xffffffffu, x >= 0 && n > 0 && t0 + end > x);
    if (in) {
      const int f = __ffs(in) - 1;
      b = b0 + f;
      return t0 + __shfl_sync(0xffffffffu, end - n, f);
    }
    t0 += __shfl_sync(0xffffffffu, end, 31);
  }
  return t0;
}
// How the tiles are cut: `n` workers, worker w from floor(w * total / n) on, none without a
// tile.
struct Cut {
  int first32;  // the lane's share of the first 32 sequences' tiles
  int total, n, q, rem;
  __device__ __forceinline__ Cut(const TreeArgs &a) {
    const int lane = threadIdx.x & 31;
    int b;
    first32 = lane < a.u.batch ? seq_tiles(a, lane) : 0;
    total = scan_tiles(a, first32, -1, b);
    n = min(a.workers, total);
    q = n > 0 ? total / n : 0;
    rem = total - q * n;
  }
  __device__ __forceinline__ int start(int w) const {
    return w < n ? w * q + w * rem / n : total;
  }
  __device__ __forceinline__ int worker(int x) const {
    return (int)((((int64_t)x + 1) * n - 1) / total);
  }
};

// A worker's range, item after item: an item is (sequence, key/value head, row tile).
struct Walk {
  int x, end;     // the next tile of the call, the range's end
  int b, nt;      // sequence, key tiles of an item
  int first;      // the item's first tile
  int hk, mt;     // key/value head, row tile
  int t;          // the segment's first key tile
  int n;          // its key tiles
  bool at_start;  // the segment begins the worker's range

  __device__ __forceinline__ void init(const TreeArgs &a, const Cut &cut, int w) {
    x = cut.start(w);
    end = cut.start(w + 1);
    at_start = true;
    if (x >= end) return;
    const int t0 = scan_tiles(a, cut.first32, x, b);
    nt = seq_tiles(a, b);
    const int item = (x - t0) / nt;
    hk = item / a.mtiles;
    mt = item - hk * a.mtiles;
    t = x - t0 - item * nt;
    first = x - t;
    n = min(nt - t, end - x);
  }
  __device__ __forceinline__ bool more() const { return x < end; }
  __device__ __forceinline__ bool whole() const { return t == 0 && n == nt; }
  __device__ __forceinline__ void next(const TreeArgs &a) {
    x += n;
    at_start = false;
    if (x >= end) return;
    t = 0;
    if (++mt == a.mtiles) {
      mt = 0;
      if (++hk == a.u.kv_heads) {
        hk = 0;
        do nt = seq_tiles(a, ++b);
        while (nt == 0);
      }
    }
    first = x;
    n = min(nt, end - x);
  }
};

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z,
                                            int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// A bounded wait of a converged warp: all its lanes learn the same outcome. `err` ends it, too.
__device__ __forceinline__ bool wait_or(uint64_t *b, uint32_t parity, volatile uint32_t *err) {
  if (__all_sync(0xffffffffu, mb_try(b, parity))) return true;
  return __all_sync(0xffffffffu, *err == 0 && mb_wait(b, parity));
}
// A product whose A operand lies in TMEM: rows by lane, two 16-bit values a column.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Descriptor of V as the N-major B operand: rows (keys, the product's K) of 128 bytes hold 64
// values of N; 8 keys further are 1024 bytes further (stride byte offset), the next 64 values
// a block of kTileT keys further (leading byte offset).
__device__ __forceinline__ uint64_t smem_desc_v(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((kTileT * 128) >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
// kind::f16 with fp32 sums, M = 128; type 1: bf16, 0: f16; b_n_major: B is N-major.
__host__ __device__ constexpr uint32_t idesc_tree(uint32_t type, int n, uint32_t b_n_major) {
  return (1u << 4) | (type << 7) | (type << 10) | (b_n_major << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileM >> 4) << 24);
}
// 64 columns of the warp's lanes; the values are there when it returns. (TMEM accesses are
// aligned: the warp has to be converged, so each stands behind a __syncwarp.)
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&r)[64]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]),
        "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]),
        "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
        "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]),
        "=f"(r[38]), "=f"(r[39]), "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]),
        "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]), "=f"(r[48]), "=f"(r[49]),
        "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
        "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]),
        "=f"(r[62]), "=f"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
      "%29, %30, %31};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}

template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
  static constexpr uint32_t kType = 1;
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <> struct Half<__half> {
  static constexpr uint32_t kType = 0;
  // P is kept 2^6 larger (at most 2^14), so that small weights stay clear of fp16's subnormals.
  static constexpr float kShift = 6.f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

template <typename T, int DP, int NS>
__global__ void __launch_bounds__(TreeCfg<DP, NS>::kThreads, NS == 1 ? 2 : 1)
    tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ TreeArgs a) {
  typedef TreeCfg<DP, NS> Cfg;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char *base = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  unsigned char *q_s = base, *k_s = base + NS * Cfg::kQ, *v_s = k_s + kStages * Cfg::kKv;
  uint64_t *bars = reinterpret_cast<uint64_t *>(base + NS * Cfg::kQ + Cfg::kRings);
  uint64_t *kfull = bars, *kempty = kfull + kStages, *vfull = kempty + kStages,
           *vempty = vfull + kStages, *sfull = vempty + kStages, *pready = sfull + 2 * NS,
           *pvdone = pready + 2 * NS, *qfull = pvdone + 2 * NS, *drain = qfull + NS;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile uint32_t *err = tmem_slot + 1;
  int32_t *parents_s = reinterpret_cast<int32_t *>(tmem_slot + 2);  // [NS][64]
  uint32_t *used_s = reinterpret_cast<uint32_t *>(parents_s + NS * TABBY_TREE_MAX_NODES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    *err = 0;
    for (int i = 0; i < kStages; i++) {
      mb_init(&kfull[i], 1);
      mb_init(&kempty[i], NS);
      mb_init(&vfull[i], 1);
      mb_init(&vempty[i], NS);
    }
    for (int i = 0; i < 2 * NS; i++) {
      mb_init(&sfull[i], 1);
      mb_init(&pready[i], 4);
      mb_init(&pvdone[i], 1);
    }
    for (int i = 0; i < NS; i++) mb_init(&qfull[i], 4);
    mb_init(drain, NS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // The previous kernel of the stream is done from here on: nothing of it waits for the TMEM
  // columns that this CTA takes.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 4 * NS + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "n"(Cfg::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be set up

  const Cut cut(a);
  Walk w;
  w.init(a, cut, blockIdx.x);

  if (warp == 4 * NS) {
    // ---- TMA producer (one lane): K tiles one ahead of V tiles, as they are consumed ----
    if (lane == 0) {
      uint32_t ik = 0, iv = 0;  // tiles loaded so far
      bool ok = true;
      auto load = [&](uint64_t *full, uint64_t *empty, unsigned char *ring, uint32_t &i,
                      const CUtensorMap *map, int tile) {
        const uint32_t s = i % kStages;
        if (!mb_wait(&empty[s], ((i / kStages) & 1u) ^ 1u)) return false;
#ifdef TABBY_CHECKS
        if (full == vfull && w.b == g_tree_checks.withhold) {
          i++;
          return true;
        }
#endif
        mb_arrive_expect(&full[s], (uint32_t)Cfg::kKv);
        for (int d = 0; d < Cfg::kBlocks; d++)
          tma_load_4d(ring + s * Cfg::kKv + d * kTileT * 128, map, d * 64, tile * kTileT, w.hk,
                      w.b, &full[s]);
        i++;
        return true;
      };
      for (; w.more() && ok; w.next(a)) {
        ok = load(kfull, kempty, k_s, ik, &map_k, w.t);
        for (int t = 0; ok && t < w.n; t++) {
          if (*err) ok = false;
          if (ok && t + 1 < w.n) ok = load(kfull, kempty, k_s, ik, &map_k, w.t + t + 1);
          if (ok) ok = load(vfull, vempty, v_s, iv, &map_v, w.t + t);
        }
      }
      if (!ok) *err = 1;
      // Every issued load lands before the CTA may end (bounded).
      for (uint32_t j = 0; j < min(ik, (uint32_t)kStages); j++)
        mb_wait(&kfull[(ik - 1 - j) % kStages], ((ik - 1 - j) / kStages) & 1u);
      for (uint32_t j = 0; j < min(iv, (uint32_t)kStages); j++)
        mb_wait(&vfull[(iv - 1 - j) % kStages], ((iv - 1 - j) / kStages) & 1u);
    }
  } else if (warp > 4 * NS) {
    // ---- MMA issuers, a warp a row tile (while one waits, the other's products run). The warp
    // goes along as one, so descriptors stay in uniform registers; an elected lane issues. K
    // steps beyond the dim multiply zeros. ----
    const int r = warp - 4 * NS - 1;
    constexpr uint32_t id_s = idesc_tree(Half<T>::kType, kTileT, 0u);
    constexpr uint32_t id_o = idesc_tree(Half<T>::kType, DP, 1u);
    const uint64_t q_desc = smem_desc(smem_addr(q_s)) + r * (Cfg::kQ >> 4);
    const uint64_t k_desc = smem_desc(smem_addr(k_s)), v_desc = smem_desc_v(smem_addr(v_s));
    const uint32_t o_tm = tmem + Cfg::kO + r * DP, s_tm = tmem + Cfg::kS + 2 * r * kTileT;
    // One barrier for the even and one for the odd tiles of each kind: who waits is never two
    // phases of a barrier behind, so a phase's parity tells it.
    uint64_t *sf = sfull + 2 * r, *pr = pready + 2 * r, *pd = pvdone + 2 * r;
    uint32_t ik = 0, iv = 0;           // K and V tiles of the worker
    uint32_t is = 0, io = 0, seg = 0;  // S tiles and O steps issued, segments begun
    bool ok = true;
    // The S tile of the segment's key tile t.
    auto issue_s = [&](int t) {
      const uint32_t s = ik % kStages;
      // S tile `is` takes the columns of P tile is - 2, which O step is - 2 has to have read.
      // (A segment's first tile finds every step done: Q's arrival stands behind them.)
      if (t > 0 && is >= 2 && !wait_or(&pd[is & 1u], ((is - 2) >> 1) & 1u, err)) return false;
      if (!wait_or(&kfull[s], (ik / kStages) & 1u, err)) return false;
      tc_fence_after();
      const uint64_t kd = k_desc + s * (Cfg::kKv >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++)
          mma_ss(s_tm + (is & 1u) * kTileT, q_desc + (kk >> 2) * (kTileM * 128 >> 4) + 2 * (kk & 3),
                 kd + (kk >> 2) * (kTileT * 128 >> 4) + 2 * (kk & 3), id_s, kk != 0);
        mma_commit(&sf[is & 1u]);
        mma_commit(&kempty[s]);
      }
      __syncwarp();
      ik++;
      is++;
      return true;
    };
    for (; w.more() && ok; w.next(a)) {
      if ((w.mt * NS + r) * kTileM >= a.mrows) {  // no such row tile: only hands the tiles back
        for (int t = 0; ok && t < w.n; t++, ik++, iv++) {
          ok = wait_or(&kfull[ik % kStages], (ik / kStages) & 1u, err);
          if (ok && lane == 0) mb_arrive(&kempty[ik % kStages]);
          ok = ok && wait_or(&vfull[iv % kStages], (iv / kStages) & 1u, err);
          if (ok && lane == 0) mb_arrive(&vempty[iv % kStages]);
        }
        continue;
      }
      ok = wait_or(&qfull[r], seg & 1u, err) && issue_s(0);
      seg++;
      for (int t = 0; ok && t < w.n; t++) {
        if (t + 1 < w.n) ok = issue_s(t + 1);
        const uint32_t s = iv % kStages;
        ok = ok && wait_or(&vfull[s], (iv / kStages) & 1u, err) &&
             wait_or(&pr[io & 1u], (io >> 1) & 1u, err);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = v_desc + s * (Cfg::kKv >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTileT / 16; kk++)
            mma_ts(o_tm, s_tm + (io & 1u) * kTileT + 8 * kk, vd + (2048 >> 4) * kk, id_o,
                   t != 0 || kk != 0);
          mma_commit(&pd[io & 1u]);
          mma_commit(&vempty[s]);
        }
        __syncwarp();
        iv++;
        io++;
#ifdef TABBY_CHECKS
        if (r == 0 && w.b == g_tree_checks.give_up) ok = false;
#endif
      }
    }
    if (!ok) *err = 1;
    // Every product is done before the tiles and TMEM go, also where a wait ran out, here or in
    // another warp: what was issued ends by itself. (Whichever issuer comes last waits for all.)
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    mb_wait(drain, 0);
    __syncwarp();
  } else {
    // ---- softmax: four warps a row tile, one row a thread ----
    const int rt = warp >> 2, r = tid & 127;  // row tile and row in it
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t o_tm = lanes + Cfg::kO + rt * DP, s_tm = lanes + Cfg::kS + 2 * rt * kTileT;
    uint64_t *pd = pvdone + 2 * rt;
    int32_t *parents = parents_s + rt * TABBY_TREE_MAX_NODES;
    uint32_t *used_bits = used_s + 2 * rt;
    unsigned char *q_t = q_s + rt * Cfg::kQ;
    const float c = a.c;
    const int dim = a.u.dim;
    uint32_t it = 0;   // tiles of the row tile
    uint32_t itv = 0;  // V tiles of the worker
    bool ok = true;
    int4 mine = make_int4(0, 0, 0, 0);  // the item that is cut first here
    for (; w.more(); itv += (uint32_t)w.n, w.next(a)) {
      const int64_t L = a.u.lengths[w.b];
      const int row = (w.mt * NS + rt) * kTileM + r;  // of the key/value head's rows
      if (row - r >= a.mrows) continue;               // no such row tile
      int32_t parent = 0;
      if (r < a.u.nodes) parent = a.u.parents[w.b * a.u.parents_stride + r];
      const int node = div_group(a, row);
      const bool real = row < a.mrows, idle = row - lane >= a.mrows;  // idle: the whole warp
      constexpr int kPieces = DP / 8;  // of 16 bytes a row
      const int row0 = row - r, piece = r % kPieces;
      // Row `y` of the tile in the 16-bit tensor `p`: the thread's piece of it.
      auto place = [&](const void *p, int y, int64_t batch, int64_t nodes, int64_t heads) {
        const int n = div_group(a, y), g = y - n * a.group;
        return const_cast<uint4 *>(reinterpret_cast<const uint4 *>(
            static_cast<const T *>(p) + w.b * batch + n * nodes +
            (int64_t)(w.hk * a.group + g) * heads + 8 * piece));
      };
      auto swizzled = [&](int y) {
        return reinterpret_cast<uint4 *>(q_t + (piece >> 3) * (kTileM * 128) + y * 128 +
                                         (((piece & 7) ^ (y & 7)) << 4));
      };
      // Q's tile: 16-byte pieces at their swizzled places, zeros beyond the rows and the dim.
      // All loads are on their way before the first is stored. (The tile's place is free: S's
      // last tile is done, and the barrier stands behind the last result's way through it.)
      asm volatile("bar.sync %0, 128;" ::"r"(1 + rt) : "memory");
      if (ok) {
        uint4 x[kPieces];
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
          const int y = row0 + r / kPieces + p * (128 / kPieces);
          x[p] = make_uint4(0, 0, 0, 0);
          if (y < a.mrows && 8 * piece < dim)
            x[p] = *place(a.u.q, y, a.u.q_batch_stride, a.u.q_node_stride, a.u.q_head_stride);
        }
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
          x[p].x = (x[p].x ^ a.q_xor) & a.q_and;
          x[p].y = (x[p].y ^ a.q_xor) & a.q_and;
          x[p].z = (x[p].z ^ a.q_xor) & a.q_and;
          x[p].w = (x[p].w ^ a.q_xor) & a.q_and;
          const int y = r / kPieces + p * (128 / kPieces);
          if (row0 + y >= a.mrows || 8 * piece >= dim) x[p] = make_uint4(0, 0, 0, 0);
          *swizzled(y) = x[p];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mb_arrive(&qfull[rt]);
      }
      // The tree: which slots the row sees, and which slots any row may see.
      if (r < a.u.nodes) parents[r] = parent;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + rt) : "memory");
      if ((warp & 3) < 2) {
        const bool in = r < a.u.nodes && L + r < a.u.entries && tree_sees(parents, r) != 0;
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        if (lane == 0) used_bits[warp & 3] = m;
      }
      unsigned long long sees = 0;
      if (real && L + node < a.u.entries) sees = tree_sees(parents, node);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + rt) : "memory");
      const unsigned long long used =
          (unsigned long long)used_bits[1] << 32 | (unsigned long long)used_bits[0];
      float m = -INFINITY, l = 0.f;  // m = c * maximum
      for (int t = 0; ok && t < w.n; t++, it++) {
        const uint32_t sb = it & 1u;
        if (!wait_or(&sfull[2 * rt + sb], (it >> 1) & 1u, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[64];
        if (!idle) tmem_ld64(s_tm + sb * kTileT, s);
        const int64_t t0 = (int64_t)(w.t + t) * kTileT;
        const bool tail = t0 + kTileT > L;  // the tile holds keys behind the context
        // A slot mask as one over the tile's keys, those of the context set.
        auto at_tile = [&](unsigned long long bits) -> unsigned long long {
          if (L >= t0) {
            const int n = (int)(L - t0);  // below 64
            return ((1ull << n) - 1) | bits << n;
          }
          return t0 - L < 64 ? bits >> (t0 - L) : 0ull;
        };
        if (tail) {
          // V's rows that no query row sees may hold anything, and 0 times NaN is NaN: they
          // become zeros before the O step.
          const uint32_t i = itv + (uint32_t)t, vs = i % kStages;
          if (!wait_or(&vfull[vs], (i / kStages) & 1u, err)) {
            ok = false;
            break;
          }
          if (!(at_tile(used) >> (r & 63) & 1)) {
#pragma unroll
            for (int d = 0; d < Cfg::kBlocks; d++)
#pragma unroll
              for (int p = 0; p < 4; p++)  // half a row a thread
                *reinterpret_cast<uint4 *>(v_s + vs * Cfg::kKv + d * kTileT * 128 +
                                           (r & 63) * 128 + (r >> 6) * 64 + 16 * p) =
                    make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (idle) {  // P's rows of this warp reach only its own rows of O, which nobody reads
          __syncwarp();
          if (lane == 0) mb_arrive(&pready[2 * rt + sb]);
          continue;
        }
        if (tail) {
          const unsigned long long see = at_tile(sees);
#pragma unroll
          for (int j = 0; j < 64; j++)
            if (!(see >> j & 1)) s[j] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int j = 4; j < 60; j += 8)
#pragma unroll
          for (int i = 0; i < 4; i++) mx[i] = max3(mx[i], s[j + 2 * i], s[j + 2 * i + 1]);
        const float top = max3(max3(mx[0], mx[1], s[60]), max3(mx[2], mx[3], s[61]),
                               fmaxf(s[62], s[63]));
        const bool rise = top * c - m > kLazy;
        if (t == 0) {
          m = top * c;
        } else if (__any_sync(0xffffffffu, rise)) {
          // O is free to change once its last step is done; this tile's is not yet issued.
          if (!wait_or(&pd[(it - 1) & 1u], ((it - 1) >> 1) & 1u, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float f = rise ? ex2_fast(m - top * c) : 1.f;
          m = rise ? top * c : m;
          l *= f;
#pragma unroll 1
          for (int d = 0; d < dim; d += 32) {
            uint32_t o[32];
            tmem_ld32(o_tm + d, o);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            tmem_st32(o_tm + d, o);
          }
        }
        const float off = (m == -INFINITY ? 0.f : m) - Half<T>::kShift;
        uint32_t p[32];
        float2 sum[2] = {};
        const float2 c2 = make_float2(c, c), off2 = make_float2(-off, -off);
#pragma unroll
        for (int j = 0; j < 32; j++) {
          float2 x = fma2(make_float2(s[2 * j], s[2 * j + 1]), c2, off2);
          x.x = ex2_fast(x.x);
          x.y = ex2_fast(x.y);
          sum[j & 1] = add2(sum[j & 1], x);
          p[j] = Half<T>::pack(x.x, x.y);
        }
        const float2 sums = add2(sum[0], sum[1]);
        l += sums.x + sums.y;
        tmem_st32(s_tm + sb * kTileT, p);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mb_arrive(&pready[2 * rt + sb]);
      }
      // The segment's result, behind its last O step.
      if (ok && !wait_or(&pd[(it - 1) & 1u], ((it - 1) >> 1) & 1u, err)) ok = false;
      if (!ok) *err = 1;
      tc_fence_after();
      const bool whole = w.whole();
      if (w.t == 0) {
        int4 c4 = make_int4(w.b, w.hk * a.mtiles + w.mt, 2 * blockIdx.x + (w.at_start ? 0 : 1), 0);
        if (!whole) c4.w = cut.worker(w.first + w.nt - 1) - (int)blockIdx.x + 1;
        if (!whole) mine = c4;
        if (a.by_item && tid == 0) a.cuts[w.b * a.u.kv_heads * a.mtiles + c4.y] = c4;
      }
      const int64_t slot = 2 * (int64_t)blockIdx.x + (w.at_start ? 0 : 1);
      const float inv = !ok ? NAN : sees == 0 ? 0.f : 1.f / l;
      if (!whole && real) a.part_ml[slot * a.prow + rt * kTileM + r] = make_float2(ok ? m : NAN, l);
      float4 *part = reinterpret_cast<float4 *>(a.part_o) + slot * (dim / 4) * a.prow +
                     rt * kTileM + r;
#pragma unroll
      for (int d = 0; d < DP; d += 32) {
        uint32_t o[32];
        tmem_ld32(o_tm + d, o);
        if (whole) {  // rows through shared memory, so that they leave whole
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
              h[e] = sees == 0 ? 0u
                               : Half<T>::pack(__uint_as_float(o[j + 2 * e]) * inv,
                                               __uint_as_float(o[j + 2 * e + 1]) * inv);
            const int pc = (d + j) / 8;
            *reinterpret_cast<uint4 *>(q_t + (pc >> 3) * (kTileM * 128) + r * 128 +
                                       (((pc & 7) ^ (r & 7)) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        } else if (real) {  // neighbouring rows lie side by side
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (d + j < dim)
              part[(d + j) / 4 * a.prow] =
                  make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]),
                              __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
        }
      }
      if (whole) {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + rt) : "memory");
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
          const int y = r / kPieces + p * (128 / kPieces);
          if (row0 + y < a.mrows && 8 * piece < dim)
            *place(a.u.out, row0 + y, a.u.out_batch_stride, a.u.out_node_stride,
                   a.u.out_head_stride) = *swizzled(y);
        }
      }
      tc_fence_before();
    }
    if (!a.by_item && tid == 0) a.cuts[blockIdx.x] = mine;
    // Sequences with nothing to attend to: zeros.
    for (int b = blockIdx.x; b < a.u.batch; b += gridDim.x) {
      if (seq_tiles(a, b) != 0) continue;
      for (int i = tid; a.by_item && i < a.u.kv_heads * a.mtiles; i += 128 * NS)
        a.cuts[b * a.u.kv_heads * a.mtiles + i] = make_int4(0, 0, 0, 0);
      const int64_t per = (int64_t)a.u.heads * dim / 8;
      for (int64_t i = tid; i < a.u.nodes * per; i += 128 * NS) {
        T *out = static_cast<T *>(a.u.out) + (int64_t)b * a.u.out_batch_stride +
                 i / per * a.u.out_node_stride + i % per / (dim / 8) * a.u.out_head_stride +
                 i % (dim / 8) * 8;
        *reinterpret_cast<uint4 *>(out) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
#ifdef TABBY_CHECKS
  if (tid == 0 && !mb_test(drain, 0)) atomicAdd(&g_tree_checks.in_flight, 1);
#endif
  if (warp == 4 * NS + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(Cfg::kTmem)
                 : "memory");
  }
}

// Joins the parts of the items that were cut between workers, with weights 2^(m_i - max m); an entry
// of `cuts` a blockIdx.x. A part's sums lie as [group of 4 values][row]: a thread takes one place
// of them, neighbours neighbouring ones, and goes through the parts; `share` threads share out the
// parts of a place.
constexpr int kJoinThreads = 256;

template <typename T, int NS>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeArgs a,
                                                                 int share) {
  __shared__ int32_t parents[TABBY_TREE_MAX_NODES];
  __shared__ float4 so[kJoinThreads];
  __shared__ float2 sml[kJoinThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = a.cuts[blockIdx.x];
  const int n = cut.w;
  if (n == 0) return;
  const int tid = threadIdx.x, places = kJoinThreads / share;
  const int first = tid / places;  // of the parts
  const int all = a.u.dim / 4 * a.prow;  // places of a part
  const int64_t b = cut.x;
  const int hk = cut.y / a.mtiles, mt = cut.y - hk * a.mtiles;
  const int64_t L = a.u.lengths[b];
  if (tid < a.u.nodes) parents[tid] = a.u.parents[b * a.u.parents_stride + tid];
  for (int p0 = blockIdx.y * places; p0 < all; p0 += gridDim.y * places) {
    const int at = p0 + tid % places, g = at / a.prow, r = at - g * a.prow;
    const int row = mt * NS * kTileM + r, node = div_group(a, row);
    const bool real = at < all && row < a.mrows;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float m1, float l1, float4 y) {
      const float m2 = fmaxf(m, m1);  // a NaN is passed over here, and kept by the sum
      const float k = m == -INFINITY ? 0.f : ex2_fast(m - m2);
      const float f = m1 == -INFINITY ? 0.f : ex2_fast(m1 - m2);
      m = m2;
      l = l * k + l1 * f;
      o = make_float4(o.x * k + y.x * f, o.y * k + y.y * f, o.z * k + y.z * f, o.w * k + y.w * f);
    };
    if (real) {
#pragma unroll 4
      for (int i = first; i < n; i += share) {
        // The parts behind the first begin their workers' ranges: those have the even slots.
        const int64_t slot = i == 0 ? cut.z : (cut.z & ~1) + 2 * i;
        const float2 ml = a.part_ml[slot * a.prow + r];
        add(ml.x, ml.y, reinterpret_cast<const float4 *>(a.part_o)[slot * all + at]);
      }
    }
    if (share > 1) {
      __syncthreads();
      so[tid] = o;
      sml[tid] = make_float2(m, l);
    }
    __syncthreads();  // the parents are there, too
    if (real && first == 0) {
      for (int i = 1; i < share; i++)
        add(sml[i * places + tid].x, sml[i * places + tid].y, so[i * places + tid]);
      const float inv = 1.f / l;
      uint2 h = make_uint2(0, 0);
      if (L + node < a.u.entries && tree_sees(parents, node) != 0)
        h = make_uint2(Half<T>::pack(o.x * inv, o.y * inv), Half<T>::pack(o.z * inv, o.w * inv));
      const int64_t head = (int64_t)hk * a.group + row - node * a.group;
      *reinterpret_cast<uint2 *>(static_cast<T *>(a.u.out) + b * a.u.out_batch_stride +
                                 node * a.u.out_node_stride + head * a.u.out_head_stride + 4 * g) =
          h;
    }
  }
}

int check_tree(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads, int32_t dim) {
  if (batch < 0) return decode_fail(TABBY_EINVAL, "tree_attention: batch must be >= 0");
  if (nodes < 1 || nodes > TABBY_TREE_MAX_NODES)
    return decode_fail(TABBY_EINVAL, "tree_attention: nodes must be in [1, %d], got %d",
                       TABBY_TREE_MAX_NODES, nodes);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65536)
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: heads (%d) must be a multiple of kv_heads (%d), at most "
                       "65536",
                       heads, kv_heads);
  if (dim < 8 || dim > TABBY_TREE_MAX_DIM || dim % 8 != 0)
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: dim must be a multiple of 8 in [8, %d], got %d",
                       TABBY_TREE_MAX_DIM, dim);
  if ((int64_t)batch * heads * nodes > INT32_MAX)
    return decode_fail(TABBY_EINVAL, "tree_attention: batch * heads * nodes exceeds 2^31 - 1");
  return TABBY_OK;
}

// [batch][head][entries][dim] as a 4-D tensor map with boxes of 64 values x kTileT entries.
bool make_cache_map(CUtensorMap *m, const void *ptr, const tabby_tree_attention_args &a,
                    int64_t batch_stride, int64_t head_stride, int64_t entry_stride) {
  EncodeTiled enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.entries, (cuuint64_t)a.kv_heads,
                              (cuuint64_t)a.batch};
  // An axis of one has no stride of its own.
  const cuuint64_t strides[3] = {2 * (cuuint64_t)(a.entries > 1 ? entry_stride : 8),
                                 2 * (cuuint64_t)(a.kv_heads > 1 ? head_stride : 8),
                                 2 * (cuuint64_t)(a.batch > 1 ? batch_stride : 8)};
  const cuuint32_t box[4] = {64, kTileT, 1, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return enc(m,
             a.dtype == TABBY_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             4, const_cast<void *>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct DeviceInfo {
  int sms = 0;
  cudaError_t err = cudaErrorUnknown;
};

// The current device's SM count, with the kernels' shared memory set; once a device.
DeviceInfo device_info() {
  constexpr int kDevices = 64;
  static DeviceInfo info[kDevices];
  static std::mutex mu;
  DeviceInfo d;
  int dev = 0;
  if ((d.err = cudaGetDevice(&dev)) != cudaSuccess) return d;
  std::lock_guard<std::mutex> lock(mu);
  if (dev < kDevices && info[dev].err == cudaSuccess) return info[dev];
  d.err = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
  auto set = [&](auto *f, size_t bytes) {
    if (d.err == cudaSuccess)
      d.err = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  };
  set(tree_kernel<__nv_bfloat16, 64, 1>, TreeCfg<64, 1>::kSmem);
  set(tree_kernel<__nv_bfloat16, 64, 2>, TreeCfg<64, 2>::kSmem);
  set(tree_kernel<__nv_bfloat16, 128, 1>, TreeCfg<128, 1>::kSmem);
  set(tree_kernel<__nv_bfloat16, 128, 2>, TreeCfg<128, 2>::kSmem);
  set(tree_kernel<__half, 64, 1>, TreeCfg<64, 1>::kSmem);
  set(tree_kernel<__half, 64, 2>, TreeCfg<64, 2>::kSmem);
  set(tree_kernel<__half, 128, 1>, TreeCfg<128, 1>::kSmem);
  set(tree_kernel<__half, 128, 2>, TreeCfg<128, 2>::kSmem);
  if (d.err == cudaSuccess && dev < kDevices) info[dev] = d;
  return d;
}

template <typename T, int DP, int NS>
cudaError_t launch_tree(const TreeArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                        cudaStream_t s) {
  typedef TreeCfg<DP, NS> Cfg;
  const cudaError_t err = launch_pdl(tree_kernel<T, DP, NS>, a.workers, Cfg::kThreads, Cfg::kSmem,
                                     s, mk, mv, a);
  if (err != cudaSuccess) return err;
  const int all = a.u.dim / 4 * a.prow;
  // Items of many parts: up to eight threads share a place's parts, as far as all of them run at
  // once. (8 sequences of 26 nodes, 40 items of 7 parts: 21.9 us a call with four, 24.7 with one; 64
  // sequences of 8 nodes, 512 items on 296 workers: 54 with one, 67 with eight.)
  int share = 1;
  while (a.by_item && share < 8 && 2 * share * a.items <= a.workers &&
         (int64_t)2 * share * a.items * all <= (int64_t)a.workers * 1024)
    share *= 2;
  const int places = kJoinThreads / share;
  return launch_pdl(tree_join_kernel<T, NS>,
                    dim3((unsigned)(a.by_item ? a.items : a.workers),
                         (unsigned)std::min((all + places - 1) / places, a.by_item ? 64 * share : 8)),
                    kJoinThreads, 0, s, a, share);
}

template <typename T>
cudaError_t launch_tree_of(const TreeArgs &a, int ns, const CUtensorMap &mk, const CUtensorMap &mv,
                           cudaStream_t s) {
  if (a.u.dim <= 64)
    return ns == 1 ? launch_tree<T, 64, 1>(a, mk, mv, s) : launch_tree<T, 64, 2>(a, mk, mv, s);
  return ns == 1 ? launch_tree<T, 128, 1>(a, mk, mv, s) : launch_tree<T, 128, 2>(a, mk, mv, s);
}

}  // namespace
}  // namespace tabby

extern "C" {

int tabby_tree_workspace_bytes(int32_t batch, int32_t nodes, int32_t heads, int32_t kv_heads,
                               int32_t dim, size_t *bytes) {
  using namespace tabby;
  const int st = check_tree(batch, nodes, heads, kv_heads, dim);
  if (st) return st;
  if (!bytes) return decode_fail(TABBY_EINVAL, "tree_attention: bytes is NULL");
  const size_t rows = (size_t)std::min<int64_t>((int64_t)nodes * (heads / kv_heads), 2 * kTileM);
  const size_t workers = (size_t)max_workers((int64_t)nodes * (heads / kv_heads));
  *bytes = workers * (2 * rows * (sizeof(float2) + (size_t)dim * sizeof(float)) + sizeof(int4));
  return TABBY_OK;
}

int tabby_tree_attention_async(int32_t device, const tabby_tree_attention_args *h_args,
                               void *stream) {
  using namespace tabby;
  if (!h_args) return decode_fail(TABBY_EINVAL, "tree_attention: args is NULL");
  const tabby_tree_attention_args a = *h_args;
  size_t need = 0;
  const int st =
      tabby_tree_workspace_bytes(a.batch, a.nodes, a.heads, a.kv_heads, a.dim, &need);
  if (st) return st;
  if (a.dtype != TABBY_BF16 && a.dtype != TABBY_F16)
    return decode_fail(TABBY_EINVAL, "tree_attention: dtype must be TABBY_BF16 or TABBY_F16");
  if (a.entries < 1) return decode_fail(TABBY_EINVAL, "tree_attention: entries must be >= 1");
  if (!(a.scale > -INFINITY && a.scale < INFINITY))
    return decode_fail(TABBY_EINVAL, "tree_attention: scale must be finite");
  if (a.batch == 0) return TABBY_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.lengths || !a.parents)
    return decode_fail(TABBY_EINVAL, "tree_attention: a required pointer is NULL");
  if (!aligned_to(a.q, 16) || !aligned_to(a.k, 16) || !aligned_to(a.v, 16) ||
      !aligned_to(a.out, 16))
    return decode_fail(TABBY_EINVAL, "tree_attention: q, k, v and out must be 16-byte aligned");
  const int64_t strides[12] = {a.q_batch_stride,   a.q_node_stride,    a.q_head_stride,
                               a.k_batch_stride,   a.k_head_stride,    a.k_entry_stride,
                               a.v_batch_stride,   a.v_head_stride,    a.v_entry_stride,
                               a.out_batch_stride, a.out_node_stride,  a.out_head_stride};
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0)
      return decode_fail(TABBY_EINVAL,
                         "tree_attention: strides must be multiples of 8 elements, >= 0");
  if ((a.batch > 1 && (a.k_batch_stride < 8 || a.v_batch_stride < 8)) ||
      (a.kv_heads > 1 && (a.k_head_stride < 8 || a.v_head_stride < 8)) ||
      (a.entries > 1 && (a.k_entry_stride < a.dim || a.v_entry_stride < a.dim)))
    return decode_fail(TABBY_EINVAL, "tree_attention: the caches' parts overlap");
  if (a.parents_stride < 0)
    return decode_fail(TABBY_EINVAL, "tree_attention: parents_stride must be >= 0");
  if (!a.workspace || a.workspace_bytes < need || !aligned_to(a.workspace, 16))
    return decode_fail(TABBY_EINVAL,
                       "tree_attention: needs a 16-byte aligned workspace of %zu bytes", need);
  DeviceScope scope(device);
  if (scope.err != cudaSuccess) return decode_cuda_fail(scope.err, "cudaSetDevice");
  const DeviceInfo info = device_info();
  if (info.err != cudaSuccess) return decode_cuda_fail(info.err, "tree_attention set-up");
  TreeArgs t = {};
  t.u = a;
  t.group = a.heads / a.kv_heads;
  t.mrows = a.nodes * t.group;
  const int ns = t.mrows > kTileM ? 2 : 1;  // row tiles that go together
  t.mtiles = (t.mrows + ns * kTileM - 1) / (ns * kTileM);
  t.prow = std::min(t.mrows, ns * kTileM);
  t.by_group = (uint32_t)((((uint64_t)1 << 32) + t.group - 1) / t.group);
  const double most = (double)a.batch * a.kv_heads * t.mtiles *
                      (((double)a.entries + kTileT - 1) / kTileT);
  if (most > 2147483647.0)
    return decode_fail(TABBY_EINVAL, "tree_attention: batch * kv_heads * entries is too large");
  const int most_workers = max_workers(t.mrows);
  t.workers = (int32_t)std::min<double>(std::min((ns == 1 ? 2 : 1) * info.sms, most_workers),
                                         std::max(1.0, most));
  t.items = a.batch * a.kv_heads * t.mtiles;  // no more than the tiles
  t.by_item = t.items <= t.workers;
  t.c = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
  t.q_xor = a.scale < 0.f ? 0x80008000u : 0u;
  t.q_and = a.scale == 0.f ? 0u : 0xffffffffu;
  t.part_o = static_cast<float *>(a.workspace);
  t.part_ml = reinterpret_cast<float2 *>(t.part_o + 2 * (size_t)most_workers * t.prow * a.dim);
  t.cuts = reinterpret_cast<int4 *>(t.part_ml + 2 * (size_t)most_workers * t.prow);
  CUtensorMap mk, mv;
  if (!make_cache_map(&mk, a.k, a, a.k_batch_stride, a.k_head_stride, a.k_entry_stride) ||
      !make_cache_map(&mv, a.v, a, a.v_batch_stride, a.v_head_stride, a.v_entry_stride))
    return decode_fail(TABBY_EINVAL, "tree_attention: the caches' layout has no tensor map");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = a.dtype == TABBY_BF16 ? launch_tree_of<__nv_bfloat16>(t, ns, mk, mv, s)
                                                : launch_tree_of<__half>(t, ns, mk, mv, s);
  if (err != cudaSuccess) return decode_cuda_fail(err, "tree_attention launch");
  return TABBY_OK;
}

#ifdef TABBY_CHECKS
// Sets the sequences whose tiles are withheld (-1: none) and gives the count of CTAs.
TABBY_API int tabby_debug_tree(int32_t withhold, int32_t give_up, int32_t *in_flight) {
  tabby::TreeChecks c;
  cudaError_t err = cudaMemcpyFromSymbol(&c, tabby::g_tree_checks, sizeof(c));
  if (err == cudaSuccess) {
    *in_flight = c.in_flight;
    c = {withhold, give_up, 0};
    err = cudaMemcpyToSymbol(tabby::g_tree_checks, &c, sizeof(c));
  }
  return (int)err;
}
#endif

}  // extern "C"
