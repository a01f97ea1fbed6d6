// Attention of a drafted tree over a key/value cache (tabby_tree_attention_async).
//
//   out[b][j][h] = sum_t softmax_t(scale q.k[t]) v[t],  t < L or t = L + (j or an ancestor)
//
// The query rows of one key/value head -- slots times grouped heads, M = nodes * group of them
// -- share its keys, so a tile of 128 rows is the M of two tensor-core products, S = Q K^T and
// O += P V, over tiles of 64 keys, and the caches are read once. Between the products the
// softmax runs in one pass: a running maximum m and sum l a row,
//   P = 2^(c S - m),  l += sum P,  and where the maximum rises: O, l *= 2^(m_old - m),
// c = scale log2(e), m = c max S. The maximum is only moved when it rises by more than 8 in the exponent
// (P then stays below 2^8), so O is rarely rescaled.
//
//   tree_kernel      one CTA a worker, two workers an SM, 192 threads. The work of a call --
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
//                    warp 5      tcgen05.mma issuer: S double-buffered (the next tile's S is
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
constexpr int kTreeThreads = 192;
constexpr int kMaxWorkers = 320;  // bounds the workspace: two a SM
constexpr float kLazy = 8.f;      // the maximum moves when it rises by more than 2^8
constexpr int kTmemCols = 256;    // O: up to 128, S: 2 x 64

// Shared memory of a worker for heads of up to DP values.
template <int DP>
struct TreeSmem {
  static constexpr int kBlocks = DP / 64;             // blocks of 64 values: one swizzle row
  static constexpr int kQ = kTileM * 128 * kBlocks;   // bytes of Q's tile
  static constexpr int kKv = kTileT * 128 * kBlocks;  // bytes of a K or V tile
  static constexpr int kStages = DP == 64 ? 4 : 2;    // tiles of each ring
  static constexpr int kRings = 2 * kStages * kKv;
  static constexpr size_t kBytes = 1024 + kQ + kRings + 1024;
};

struct TreeArgs {
  tabby_tree_attention_args u;
  int32_t group;    // heads a key/value head
  int32_t mrows;    // query rows of a key/value head
  int32_t mtiles;   // row tiles of a key/value head
  int32_t workers;  // CTAs the key tiles are cut over
  int32_t prow;     // rows a part holds: min(mrows, 128)
  float c;          // |scale| log2(e), 1 where scale is 0
  uint32_t q_xor;   // flips the signs of Q's values where scale is negative
  uint32_t q_and;   // 0 where scale is 0
  float *part_o;    // [2 * workers][prow][dim]: unscaled sums
  float2 *part_ml;  // [2 * workers][prow]: m, sum
};

// Key tiles of one (head, row tile) of a sequence; 0: nothing to attend to.
__device__ __forceinline__ int64_t seq_tiles(const TreeArgs &a, int64_t b) {
  const int64_t L = a.u.lengths[b];
  if (L < 0 || L >= a.u.entries) return 0;
  const int64_t n = min(L + a.u.nodes, (int64_t)a.u.entries);
  return (n + kTileT - 1) / kTileT;
}
// All key tiles of the call (warp-uniform result; all lanes call).
__device__ __forceinline__ int64_t all_tiles(const TreeArgs &a) {
  int64_t n = 0;
  for (int64_t b = threadIdx.x & 31; b < a.u.batch; b += 32) n += seq_tiles(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.u.kv_heads * a.mtiles;
}
// Where the tile `x` of the call lies: its sequence and the number of tiles before it (all
// lanes call; x must be below all_tiles).
__device__ __forceinline__ void find_tile(const TreeArgs &a, int64_t x, int64_t &b, int64_t &t0) {
  const int lane = threadIdx.x & 31;
  const int64_t per = (int64_t)a.u.kv_heads * a.mtiles;
  t0 = 0;
  for (int64_t b0 = 0; b0 < a.u.batch; b0 += 32) {
    const int64_t n = b0 + lane < a.u.batch ? seq_tiles(a, b0 + lane) * per : 0;
    int64_t end = n;  // inclusive prefix sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += y;
    }
    const unsigned in = __ballot_sync(0xffffffffu, n > 0 && t0 + end > x);
    if (in) {
      const int f = __ffs(in) - 1;
      b = b0 + f;
      t0 += __shfl_sync(0xffffffffu, end - n, f);
      return;
    }
    t0 += __shfl_sync(0xffffffffu, end, 31);
  }
  b = 0;  // not reached
}
// How the tiles are cut: `n` workers, worker w from w * total / n on, none without a tile.
struct Cut {
  int64_t total, n;
  __device__ __forceinline__ Cut(const TreeArgs &a)
      : total(all_tiles(a)), n(min((int64_t)a.workers, total)) {}
  __device__ __forceinline__ int64_t start(int64_t w) const { return w < n ? w * total / n : total; }
  __device__ __forceinline__ int64_t worker(int64_t x) const { return ((x + 1) * n - 1) / total; }
};

// A worker's range, item after item: an item is (sequence, key/value head, row tile).
struct Walk {
  int64_t x, end;      // the next tile of the call, the range's end
  int64_t b, nt;       // sequence, key tiles of an item
  int32_t hk, mt;      // key/value head, row tile
  int64_t t;           // the segment's first key tile
  int64_t n;           // its key tiles
  bool at_start;       // the segment begins the worker's range

  __device__ __forceinline__ void init(const TreeArgs &a, const Cut &cut, int w) {
    x = cut.start(w);
    end = cut.start(w + 1);
    at_start = true;
    if (x >= end) return;
    int64_t t0;
    find_tile(a, x, b, t0);
    nt = seq_tiles(a, b);
    const int64_t item = (x - t0) / nt;
    hk = (int32_t)(item / a.mtiles);
    mt = (int32_t)(item % a.mtiles);
    t = (x - t0) % nt;
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
// 64 columns of the warp's lanes; the values are there when it returns.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&r)[64]) {
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

template <typename T, int DP>
__global__ void __launch_bounds__(kTreeThreads, 2)
    tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ TreeArgs a) {
  typedef TreeSmem<DP> Smem;
  constexpr int kStages = Smem::kStages;
  constexpr uint32_t kO = 0, kS = DP;  // TMEM columns of O and of the two S tiles
  extern __shared__ unsigned char smem_dyn[];
  unsigned char *base = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  unsigned char *q_s = base, *k_s = base + Smem::kQ, *v_s = k_s + kStages * Smem::kKv;
  uint64_t *bars = reinterpret_cast<uint64_t *>(base + Smem::kQ + Smem::kRings);
  uint64_t *kfull = bars, *kempty = kfull + kStages, *vfull = kempty + kStages,
           *vempty = vfull + kStages, *sfull = vempty + kStages, *pready = sfull + 2,
           *pvdone = pready + 2, *qfull = pvdone + 1, *drain = qfull + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile uint32_t *err = tmem_slot + 1;
  int32_t *parents = reinterpret_cast<int32_t *>(tmem_slot + 2);                 // [64]
  uint32_t *used_bits = reinterpret_cast<uint32_t *>(parents + TABBY_TREE_MAX_NODES);  // [2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    *err = 0;
    for (int i = 0; i < kStages; i++) {
      mb_init(&kfull[i], 1);
      mb_init(&kempty[i], 1);
      mb_init(&vfull[i], 1);
      mb_init(&vempty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mb_init(&sfull[i], 1);
      mb_init(&pready[i], 4);
    }
    mb_init(pvdone, 1);
    mb_init(qfull, 4);
    mb_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // The previous kernel of the stream is done from here on: nothing of it waits for the TMEM
  // columns that this CTA takes.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "n"(kTmemCols)
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

  if (warp == 4) {
    // ---- TMA producer (one lane): K tiles one ahead of V tiles, as they are consumed ----
    if (lane == 0) {
      uint32_t ik = 0, iv = 0;  // tiles loaded so far
      bool ok = true;
      auto load = [&](uint64_t *full, uint64_t *empty, unsigned char *ring, uint32_t &i,
                      const CUtensorMap *map, int64_t tile) {
        const uint32_t s = i % kStages;
        if (!mb_wait(&empty[s], ((i / kStages) & 1u) ^ 1u)) return false;
        mb_arrive_expect(&full[s], (uint32_t)Smem::kKv);
        for (int d = 0; d < Smem::kBlocks; d++)
          tma_load_4d(ring + s * Smem::kKv + d * kTileT * 128, map, d * 64, (int)(tile * kTileT),
                      w.hk, (int)w.b, &full[s]);
        i++;
        return true;
      };
      for (; w.more() && ok; w.next(a)) {
        ok = load(kfull, kempty, k_s, ik, &map_k, w.t);
        for (int64_t t = 0; ok && t < w.n; t++) {
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
  } else if (warp == 5) {
    // ---- MMA issuer: the warp goes along as one (so descriptors stay in uniform registers),
    // an elected lane issues. K steps beyond the dim multiply zeros. ----
    constexpr uint32_t id_s = idesc_tree(Half<T>::kType, kTileT, 0u);
    constexpr uint32_t id_o = idesc_tree(Half<T>::kType, DP, 1u);
    const uint64_t q_desc = smem_desc(smem_addr(q_s)), k_desc = smem_desc(smem_addr(k_s));
    const uint64_t v_desc = smem_desc_v(smem_addr(v_s));  // in units of 16 bytes from here on
    uint32_t is = 0, io = 0, seg = 0;  // S tiles and O steps issued, segments begun
    bool ok = true;
    auto issue_s = [&](int64_t t) {
      const uint32_t s = is % kStages;
      // S tile `is` takes the columns of P tile is - 2, which O step is - 2 has to have read.
      // (A segment's first tile finds every step done: Q's arrival stands behind them.)
      if (t > 0 && is >= 2 && !wait_or(pvdone, (is - 2) & 1u, err)) return false;
      if (!wait_or(&kfull[s], (is / kStages) & 1u, err)) return false;
      tc_fence_after();
      const uint32_t d = tmem + kS + (is & 1u) * kTileT;
      const uint64_t kd = k_desc + s * (Smem::kKv >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; kk++)
          mma_ss(d, q_desc + (kk >> 2) * (kTileM * 128 >> 4) + 2 * (kk & 3),
                 kd + (kk >> 2) * (kTileT * 128 >> 4) + 2 * (kk & 3), id_s, kk != 0);
        mma_commit(&kempty[s]);
        mma_commit(&sfull[is & 1u]);
      }
      __syncwarp();
      is++;
      return true;
    };
    for (; w.more() && ok; w.next(a), seg++) {
      ok = wait_or(qfull, seg & 1u, err) && issue_s(0);
      for (int64_t t = 0; ok && t < w.n; t++) {
        if (ok && t + 1 < w.n) ok = issue_s(t + 1);
        const uint32_t s = io % kStages;
        ok = ok && wait_or(&vfull[s], (io / kStages) & 1u, err) &&
             wait_or(&pready[io & 1u], (io >> 1) & 1u, err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t p = tmem + kS + (io & 1u) * kTileT;
        const uint64_t vd = v_desc + s * (Smem::kKv >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTileT / 16; kk++)
            mma_ts(tmem + kO, p + 8 * kk, vd + (2048 >> 4) * kk, id_o, t != 0 || kk != 0);
          mma_commit(&vempty[s]);
          mma_commit(pvdone);
        }
        __syncwarp();
        io++;
      }
    }
    if (!ok) *err = 1;
    if (elect_one()) mma_commit(drain);  // every product is done before TMEM goes
    __syncwarp();
    wait_or(drain, 0, err);
  } else {
    // ---- softmax, one row a thread ----
    const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
    const float c = a.c;
    const int dim = a.u.dim;
    uint32_t it = 0;  // tiles seen
    bool ok = true;
    for (; w.more(); w.next(a)) {
      const int64_t L = a.u.lengths[w.b];
      const int row = w.mt * kTileM + tid;       // of the key/value head's rows
      const int node = row / a.group;
      const int64_t head = w.hk * a.group + row % a.group;
      const bool real = row < a.mrows;
      // The tree: which slots the row sees, and which slots any row may see.
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (tid < a.u.nodes) parents[tid] = a.u.parents[w.b * a.u.parents_stride + tid];
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (warp < 2) {
        const bool in = tid < a.u.nodes && L + tid < a.u.entries && tree_sees(parents, tid) != 0;
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        if (lane == 0) used_bits[warp] = m;
      }
      unsigned long long sees = 0;
      if (real && L + node < a.u.entries) sees = tree_sees(parents, node);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      const unsigned long long used =
          (unsigned long long)used_bits[1] << 32 | (unsigned long long)used_bits[0];
      // Q's tile: 16-byte pieces at their swizzled places, zeros beyond the rows and the dim.
      if (ok) {
        const T *q = static_cast<const T *>(a.u.q) + w.b * a.u.q_batch_stride +
                     node * a.u.q_node_stride + head * a.u.q_head_stride;
#pragma unroll
        for (int p = 0; p < DP / 8; p++) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (real && 8 * p < dim) {
            x = *reinterpret_cast<const uint4 *>(q + 8 * p);
            x.x = (x.x ^ a.q_xor) & a.q_and;
            x.y = (x.y ^ a.q_xor) & a.q_and;
            x.z = (x.z ^ a.q_xor) & a.q_and;
            x.w = (x.w ^ a.q_xor) & a.q_and;
          }
          *reinterpret_cast<uint4 *>(q_s + (p >> 3) * (kTileM * 128) + tid * 128 +
                                     (((p & 7) ^ (tid & 7)) << 4)) = x;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mb_arrive(qfull);
      }
      float m = -INFINITY, l = 0.f;  // m = c * maximum
      for (int64_t t = 0; ok && t < w.n; t++, it++) {
        const uint32_t sb = it & 1u;
        if (!wait_or(&sfull[sb], (it >> 1) & 1u, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[64];
        tmem_ld64(lanes + kS + sb * kTileT, s);
        const int64_t t0 = (w.t + t) * kTileT;
        if (t0 + kTileT > L) {
          // Keys behind the context: those the row sees. V's rows that no row sees may hold
          // anything, and 0 times NaN is NaN: they become zeros.
          auto place = [&](unsigned long long bits) -> unsigned long long {
            if (L >= t0) {
              const int n = (int)(L - t0);  // below 64
              return (1ull << n) - 1 | bits << n;
            }
            return t0 - L < 64 ? bits >> (t0 - L) : 0ull;
          };
          const unsigned long long see = place(sees), any = place(used);
#pragma unroll
          for (int j = 0; j < 64; j++)
            if (!(see >> j & 1)) s[j] = -INFINITY;
          const uint32_t vs = it % kStages;
          if (!wait_or(&vfull[vs], (it / kStages) & 1u, err)) {
            ok = false;
            break;
          }
          if (!(any >> (tid & 63) & 1)) {
#pragma unroll
            for (int d = 0; d < Smem::kBlocks; d++)
#pragma unroll
              for (int p = 0; p < 4; p++)  // half a row a thread
                *reinterpret_cast<uint4 *>(v_s + vs * Smem::kKv + d * kTileT * 128 +
                                           (tid & 63) * 128 + (tid >> 6) * 64 + 16 * p) =
                    make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int j = 4; j < 64; j++) mx[j & 3] = fmaxf(mx[j & 3], s[j]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool rise = top * c - m > kLazy;
        if (t == 0) {
          m = top * c;
        } else if (__any_sync(0xffffffffu, rise)) {
          // O is free to change once its last step is done (the one before stood before this S
          // tile); this tile's is not yet issued.
          if (!wait_or(pvdone, (it - 1) & 1u, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float f = rise ? ex2_fast(m - top * c) : 1.f;
          m = rise ? top * c : m;
          l *= f;
#pragma unroll 1
          for (int d = 0; d < 16 * ((dim + 15) / 16); d += 32) {
            uint32_t o[32];
            tmem_ld32(lanes + kO + d, o);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            tmem_st32(lanes + kO + d, o);
          }
        }
        const float off = (m == -INFINITY ? 0.f : m) - Half<T>::kShift;
        uint32_t p[32];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 32; j++) {
          const float x = ex2_fast(fmaf(s[2 * j], c, -off));
          const float y = ex2_fast(fmaf(s[2 * j + 1], c, -off));
          sum[(2 * j) & 3] += x;
          sum[(2 * j + 1) & 3] += y;
          p[j] = Half<T>::pack(x, y);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st32(lanes + kS + sb * kTileT, p);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mb_arrive(&pready[sb]);
      }
      // The segment's result. S tile it - 1 stood behind O step it - 3: the last two are waited
      // for one after the other (a parity alone does not tell a step from the one two before).
      if (ok && w.n > 1 && !wait_or(pvdone, (it - 2) & 1u, err)) ok = false;
      if (ok && !wait_or(pvdone, (it - 1) & 1u, err)) ok = false;
      if (!ok) *err = 1;
      tc_fence_after();
      const bool whole = w.whole();
      const int64_t slot = 2 * (int64_t)blockIdx.x + (w.at_start ? 0 : 1);
      const float inv = !ok ? NAN : 1.f / l;
      T *out = static_cast<T *>(a.u.out) + w.b * a.u.out_batch_stride +
               node * a.u.out_node_stride + head * a.u.out_head_stride;
      float *part = a.part_o + (slot * a.prow + tid) * dim;
      if (!whole && real) a.part_ml[slot * a.prow + tid] = make_float2(ok ? m : NAN, l);
#pragma unroll
      for (int d = 0; d < DP; d += 32) {
        uint32_t o[32];
        if (ok) {
          tmem_ld32(lanes + kO + d, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) o[j] = 0x7fffffffu;
        }
        if (!real) continue;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (d + j >= dim) continue;
          if (whole) {
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
              h[e] = sees == 0 ? 0u
                               : Half<T>::pack(__uint_as_float(o[j + 2 * e]) * inv,
                                               __uint_as_float(o[j + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4 *>(out + d + j) = make_uint4(h[0], h[1], h[2], h[3]);
          } else {
            *reinterpret_cast<uint4 *>(part + d + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            *reinterpret_cast<uint4 *>(part + d + j + 4) =
                make_uint4(o[j + 4], o[j + 5], o[j + 6], o[j + 7]);
          }
        }
      }
      tc_fence_before();
    }
    // Sequences with nothing to attend to: zeros.
    for (int64_t b = blockIdx.x; b < a.u.batch; b += gridDim.x) {
      if (seq_tiles(a, b) != 0) continue;
      const int64_t per = (int64_t)a.u.heads * dim / 8;
      for (int64_t i = tid; i < a.u.nodes * per; i += 128) {
        T *out = static_cast<T *>(a.u.out) + b * a.u.out_batch_stride +
                 i / per * a.u.out_node_stride + i % per / (dim / 8) * a.u.out_head_stride +
                 i % (dim / 8) * 8;
        *reinterpret_cast<uint4 *>(out) = make_uint4(0, 0, 0, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(kTmemCols)
                 : "memory");
  }
}

// Joins the parts of the item that the start of worker blockIdx.x's range cuts first: weights
// 2^(m_i - max m) for the parts' sums. A warp takes a row, its lanes 4 values each.
template <typename T>
__global__ void __launch_bounds__(128) tree_join_kernel(const __grid_constant__ TreeArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Cut cut(a);
  const int64_t w = blockIdx.x, x = cut.start(w);
  if (w == 0 || x >= cut.total) return;
  int64_t b, t0;
  find_tile(a, x, b, t0);
  const int64_t nt = seq_tiles(a, b), item = (x - t0) / nt;
  const int64_t first = t0 + item * nt;  // the item's first tile
  const int64_t w0 = cut.worker(first), w1 = cut.worker(first + nt - 1);
  if (w != w0 + 1) return;  // not the first cut of an item
  const int hk = (int)(item / a.mtiles), mt = (int)(item % a.mtiles);
  __shared__ int32_t parents[TABBY_TREE_MAX_NODES];
  if ((int)threadIdx.x < a.u.nodes)
    parents[threadIdx.x] = a.u.parents[b * a.u.parents_stride + threadIdx.x];
  __syncthreads();
  const int64_t L = a.u.lengths[b];
  const int rows = min(a.mrows - mt * kTileM, kTileM);
  for (int r = blockIdx.y * 4 + warp; r < rows; r += gridDim.y * 4) {
    const int row = mt * kTileM + r, node = row / a.group;
    const int64_t head = (int64_t)hk * a.group + row % a.group;
    const bool seen = L + node < a.u.entries && tree_sees(parents, node) != 0;
    // Every part but the first begins its worker's range.
    auto slot = [&](int64_t i) {
      return 2 * i + (i == w0 && cut.start(w0) != first ? 1 : 0);
    };
    float m = -INFINITY;
    bool bad = false;
    for (int64_t i = w0 + lane; i <= w1; i += 32) {
      const float y = a.part_ml[slot(i) * a.prow + r].x;
      bad |= isnan(y);
      m = fmaxf(m, y);
    }
    bad = __any_sync(0xffffffffu, bad);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i = w0; i <= w1; i++) {
      const float2 ml = a.part_ml[slot(i) * a.prow + r];
      const float f = ml.x == -INFINITY ? 0.f : ex2_fast(ml.x - m);
      l += f * ml.y;
      if (4 * lane < a.u.dim) {
        const float4 y = *reinterpret_cast<const float4 *>(
            a.part_o + (slot(i) * a.prow + r) * a.u.dim + 4 * lane);
        o[0] += f * y.x;
        o[1] += f * y.y;
        o[2] += f * y.z;
        o[3] += f * y.w;
      }
    }
    if (4 * lane < a.u.dim) {
      const float inv = bad ? NAN : 1.f / l;
      uint2 h = make_uint2(0, 0);
      if (seen)
        h = make_uint2(Half<T>::pack(o[0] * inv, o[1] * inv), Half<T>::pack(o[2] * inv, o[3] * inv));
      *reinterpret_cast<uint2 *>(static_cast<T *>(a.u.out) + b * a.u.out_batch_stride +
                                 node * a.u.out_node_stride + head * a.u.out_head_stride +
                                 4 * lane) = h;
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
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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
  auto set = [](const void *f, size_t bytes) {
    return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  };
  if ((d.err = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev)) ==
          cudaSuccess &&
      (d.err = set((const void *)tree_kernel<__nv_bfloat16, 64>, TreeSmem<64>::kBytes)) ==
          cudaSuccess &&
      (d.err = set((const void *)tree_kernel<__nv_bfloat16, 128>, TreeSmem<128>::kBytes)) ==
          cudaSuccess &&
      (d.err = set((const void *)tree_kernel<__half, 64>, TreeSmem<64>::kBytes)) == cudaSuccess &&
      (d.err = set((const void *)tree_kernel<__half, 128>, TreeSmem<128>::kBytes)) ==
          cudaSuccess &&
      dev < kDevices)
    info[dev] = d;
  return d;
}

template <typename T>
cudaError_t launch_tree(const TreeArgs &a, const CUtensorMap &mk, const CUtensorMap &mv,
                        cudaStream_t s) {
  cudaError_t err =
      a.u.dim <= 64
          ? launch_pdl(tree_kernel<T, 64>, a.workers, kTreeThreads, TreeSmem<64>::kBytes, s, mk,
                       mv, a)
          : launch_pdl(tree_kernel<T, 128>, a.workers, kTreeThreads, TreeSmem<128>::kBytes, s, mk,
                       mv, a);
  if (err != cudaSuccess) return err;
  return launch_pdl(tree_join_kernel<T>, dim3(a.workers, (a.prow + 15) / 16), 128, 0, s, a);
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
  const size_t rows = (size_t)std::min<int64_t>((int64_t)nodes * (heads / kv_heads), kTileM);
  *bytes = 2 * (size_t)kMaxWorkers * rows * (sizeof(float2) + (size_t)dim * sizeof(float));
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
  t.mtiles = (t.mrows + kTileM - 1) / kTileM;
  t.prow = std::min(t.mrows, kTileM);
  const double most = (double)a.batch * a.kv_heads * t.mtiles *
                      (((double)a.entries + kTileT - 1) / kTileT);
  t.workers = (int32_t)std::min<double>(std::min(2 * info.sms, kMaxWorkers), std::max(1.0, most));
  t.c = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
  t.q_xor = a.scale < 0.f ? 0x80008000u : 0u;
  t.q_and = a.scale == 0.f ? 0u : 0xffffffffu;
  t.part_o = static_cast<float *>(a.workspace);
  t.part_ml = reinterpret_cast<float2 *>(t.part_o + 2 * (size_t)kMaxWorkers * t.prow * a.dim);
  CUtensorMap mk, mv;
  if (!make_cache_map(&mk, a.k, a, a.k_batch_stride, a.k_head_stride, a.k_entry_stride) ||
      !make_cache_map(&mv, a.v, a, a.v_batch_stride, a.v_head_stride, a.v_entry_stride))
    return decode_fail(TABBY_EINVAL, "tree_attention: the caches' layout has no tensor map");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = a.dtype == TABBY_BF16 ? launch_tree<__nv_bfloat16>(t, mk, mv, s)
                                                : launch_tree<__half>(t, mk, mv, s);
  if (err != cudaSuccess) return decode_cuda_fail(err, "tree_attention launch");
  return TABBY_OK;
}

}  // extern "C"
