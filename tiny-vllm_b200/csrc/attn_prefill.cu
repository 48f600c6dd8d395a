// Attention of whole prompts: packed sequences, causal, grouped heads, keys packed or in pages.
//
// o_i = sum_j 2^(t_ij - top_i) v_j / sum_j 2^(t_ij - top_i),  t_ij = scale log2(e) q_i . k_j,  in one pass over the keys with a
// running maximum and sum.
//
// Bound by the tensor cores and, at the same rate, by the exponentials: a tile of 128 rows x 128 keys of D = 128 is 2 x 128^3
// multiply-adds (1024 cycles) and 128^2 exponentials (1024 cycles at 16 a cycle).  So a CTA works on two tiles of rows
// in turn: while the tensor cores multiply for one, the other's four warps take their exponentials.
//
// A row of a tile is one head of one query: the G heads that share a key head stand side by side, 128 / G queries
// to a tile, so keys are loaded once for all of them and short sequences of many heads still fill their rows.
// Tensor memory (512 columns): S0, S1 (128 x 128 fp32 scores; the weights P, 16-bit, take their first half over),
// O0, O1 (128 x D sums).  Shared memory: both Q tiles and a ring of K and V tiles.
//   S_t = Q_t K^T    both operands in shared memory
//   O_t += P_t V      P from tensor memory, V as rows of keys
// Warps: 0-3 and 4-7 softmax of tile 0 and 1, a row a thread; 8 issues the products; 9 brings Q, K and V; 10 and 11
// only give their registers up.
// Keys go from the last tile, where the mask is, to the first.  The running maximum is raised, and O_t rescaled in place, only
// when a score exceeds it by more than 8 (weights reach 2^8 at most, rounded with the same relative error).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "attn.h"
#include "attn_device.cuh"
#include "common.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

constexpr int kRows = 128;                        // of a tile of queries, and keys of a tile of keys
constexpr int kThreads = 384;                    // three warpgroups; 168 registers a thread at launch
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "registers");
constexpr int kCtrlBytes = 512;
constexpr int kTmemCols = 512;
constexpr uint32_t kColO = 256;
constexpr float kLazy = 8.f;

template <int D>
constexpr int stages() { return D == 128 ? 5 : 8; }
template <int D>
constexpr int smem_bytes() { return (2 + stages<D>()) * kRows * D * 2 + kCtrlBytes; }

struct PrefillParams {
  void* out;
  const int32_t *cu_q, *cu_k, *tables;
  int64_t table_stride;
  int tokens, key_tokens, sequences, heads, kv_heads, group, dim, pages, page_size, table_width;
  int tile_tokens;      // queries of a tile: 128 / group
  int box_rows;
  int causal;
  float scale_log2;
  int* status;
};

// The queries of one sequence that a CTA works on, and the sequence's keys.
struct Item {
  int b, n, m;          // sequence, its queries and keys
  int first;            // first query of the CTA in its sequence
  int row0, key0;       // where the sequence begins in q and in packed keys
};

__device__ __forceinline__ int begin_of(const PrefillParams& p, int b) { return min(max(p.cu_q[b], 0), p.tokens); }
__device__ __forceinline__ int queries_of(const PrefillParams& p, int b) {
  return max(min(p.cu_q[b + 1], p.tokens) - begin_of(p, b), 0);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                    const __grid_constant__ CUtensorMap tmap_v, const PrefillParams p) {
  constexpr int kHalves = D / 64;
  constexpr int kHalfBytes = kRows * 128;
  constexpr int kTileBytes = kRows * D * 2;
  constexpr int kStages = stages<D>();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + 2 * kTileBytes;
  uint8_t* ctrl = ring + kStages * kTileBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(ctrl);   // [stages] a K or V tile is there
  uint64_t* free_bar = full_bar + kStages;                  // [4], in turn: products up to a step are done
  uint64_t* s_bar = free_bar + 4;                           // [2] scores of a tile are there
  uint64_t* p_bar = s_bar + 2;                              // [2][2] its weights are, of half of the keys
  uint64_t* o_bar = p_bar + 4;                              // all products are done
  uint64_t* q_bar = o_bar + 1;
  uint64_t* tail_bar = q_bar + 1;                           // the last V tile, before its end is zeroed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);        // [warps]
  Item* s_item = reinterpret_cast<Item*>(scan + kThreads / 32);
  static_assert(8 * (kStages + 13) + 8 + kThreads / 8 + sizeof(Item) <= kCtrlBytes, "control words");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = ptx::smem_u32(smem), ring_base = smem_base + 2 * kTileBytes;
  if ((smem_base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 0x200);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(ptx::smem_u32(full_bar + s), 1);
    for (int e = 0; e < 4; ++e) ptx::mbar_init(ptx::smem_u32(free_bar + e), 1);
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(s_bar + t), 1);
      ptx::mbar_init(ptx::smem_u32(p_bar + 2 * t), 4);
      ptx::mbar_init(ptx::smem_u32(p_bar + 2 * t + 1), 4);
    }
    ptx::mbar_init(ptx::smem_u32(o_bar), 1);
    ptx::mbar_init(ptx::smem_u32(q_bar), 1);
    ptx::mbar_init(ptx::smem_u32(tail_bar), 1);
    *abort_flag = 0;
    s_item->b = -1;
    ptx::fence_mbar_init();
    ptx::tma_prefetch_desc(&tmap_q);
    ptx::tma_prefetch_desc(&tmap_k);
    ptx::tma_prefetch_desc(&tmap_v);
  }
  if (warp == 8) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();

  // Which queries: items of two tiles, sequence by sequence; the last one, with the most keys, is taken first.
  const int kv = blockIdx.x % p.kv_heads, per_item = 2 * p.tile_tokens;
  {
    const int per = (p.sequences + kThreads - 1) / kThreads, b0 = threadIdx.x * per, b1 = min(b0 + per, p.sequences);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += (queries_of(p, b) + per_item - 1) / per_item;
    int upto = mine;
    for (int x = 1; x < 32; x *= 2) {
      const int o = __shfl_up_sync(~0u, upto, x);
      if (lane >= x) upto += o;
    }
    if (lane == 31) scan[warp] = upto;
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    int total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) upto += total;
      total += scan[w];
    }
    const int item = total - 1 - static_cast<int>(blockIdx.x) / p.kv_heads;
    int first = upto - mine;
    if (item >= first && item < upto) {      // one thread, or none
      int b = b0, n;
      while (true) {
        n = queries_of(p, b);
        const int items = (n + per_item - 1) / per_item;
        if (item < first + items) break;
        first += items;
        ++b;
      }
      Item it;
      it.b = b, it.n = n, it.first = (item - first) * per_item, it.row0 = begin_of(p, b);
      it.key0 = p.cu_k[b];
      int64_t m = p.cu_k[b + 1] - static_cast<int64_t>(it.key0);
      if (p.page_size > 0) m = min(m, static_cast<int64_t>(p.table_width) * p.page_size);
      else m = it.key0 < 0 ? 0 : min(m, static_cast<int64_t>(p.key_tokens) - it.key0);
      it.m = static_cast<int>(min(max(m, int64_t{0}), static_cast<int64_t>(INT_MAX - kRows)));
      *s_item = it;
    }
    __syncthreads();
  }
  const Item it = *s_item;
  const uint32_t tmem_base = *tmem_slot;      // all columns: 0, which the products' constants rely on
  if (tmem_base != 0 && threadIdx.x == 0) atomicCAS(p.status, 0, 0x200);

  if (it.b >= 0 && tmem_base == 0) {
    // Keys that query i sees: [0, seen(i)).
    const auto seen = [&](int i) { return max(0, p.causal ? min(it.m, i + 1 + it.m - it.n) : it.m); };
    int tiles[2], steps = 0;      // of keys
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int from = it.first + t * p.tile_tokens, to = min(from + p.tile_tokens, it.n);
      tiles[t] = from < to ? (seen(to - 1) + kRows - 1) / kRows : 0;
      steps = max(steps, tiles[t]);
    }
    const int skip[2] = {steps - tiles[0], steps - tiles[1]};     // the last tiles of keys that a tile of rows does not see
    const bool tail = steps * kRows > it.m;                        // the last tile of keys is not full

    if (warp == 9) {
      ptx::lower_registers<kOtherRegs>();
      // ---------------------------------------------------------------- Q, K and V
      bool alive = true;
      if (lane == 0 && steps > 0) {
        const uint32_t bar = ptx::smem_u32(q_bar), rows = p.tile_tokens * p.group * 128;
        ptx::mbar_arrive_expect_tx(bar, rows * kHalves * ((tiles[0] > 0) + (tiles[1] > 0)));
        for (int t = 0; t < 2; ++t)
          for (int h = 0; h < kHalves && tiles[t] > 0; ++h)
            ptx::tma_load_4d(smem_base + t * kTileBytes + h * kHalfBytes, &tmap_q, bar, h * 64, 0, kv,
                             it.row0 + it.first + t * p.tile_tokens);
      }
      __syncwarp();
      const int boxes = kRows / p.box_rows;
      const int32_t* table = p.page_size > 0 ? p.tables + it.b * p.table_stride : nullptr;
      int stage = 0, freed = 0, page = 0;
      uint32_t phase = 0;
      for (int s = 0; s < steps; ++s) {
        const int begin = (steps - 1 - s) * kRows;
        int at = it.key0 + begin, held = 1, mine = 0;
        if (p.page_size > 0) {
          // pages of the next 32 boxes at a time, from the last key backwards
          if (s * boxes % 32 == 0) {
            const int64_t pos = static_cast<int64_t>(steps) * kRows - static_cast<int64_t>(s * boxes + lane + 1) * p.box_rows;
            page = 0;
            if (pos >= 0 && pos < it.m) {
              page = table[pos / p.page_size];
              if (page < 0 || page >= p.pages) {
                atomicCAS(p.status, 0, 0xa01);
                page = p.pages;                                     // outside: the copy brings zeros
              }
            }
          }
          mine = __shfl_sync(~0u, page, (s * boxes + boxes - 1 - lane) & 31);
          at = (begin + lane * p.box_rows) % p.page_size;
          held = min(boxes, (it.m - begin + p.box_rows - 1) / p.box_rows);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          // Tile n = 2 s + x takes the place of tile n - kStages: the first key tile is free with the first signal, and the
          // values of step e - 1 and the keys of step e with signal e.
          const int need = (2 * s + x - kStages + 1) >> 1;
          for (; freed <= need; ++freed)
            if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(free_bar + (freed & 3)), (freed >> 2) & 1, abort_flag));
          const uint32_t bar = ptx::smem_u32(x == 1 && s == 0 && tail ? tail_bar : full_bar + stage);
          if (lane == 0 && alive) ptx::mbar_arrive_expect_tx(bar, held * p.box_rows * D * 2);
          __syncwarp();
          if (lane < held && alive)
            for (int h = 0; h < kHalves; ++h)
              ptx::tma_load_4d(ring_base + stage * kTileBytes + h * kHalfBytes + lane * p.box_rows * 128,
                               x == 0 ? &tmap_k : &tmap_v, bar, h * 64, kv, at, mine);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
        if (*abort_flag != 0) ptx::drain_ring(full_bar, kStages, stage, phase);
        if (*abort_flag != 0) ptx::drain_ring(q_bar, steps > 0 ? 1 + tail : 0, 2, 0);      // and the tail's barrier
      }
    } else if (warp == 8) {
      ptx::lower_registers<kOtherRegs>();
      // ---------------------------------------------------------------- products
      // The whole warp walks and one lane issues.
      constexpr uint32_t ab = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc_s = ptx::umma_idesc(1u, ab, kRows, kRows);
      const uint32_t idesc_o = ptx::umma_idesc(1u, ab, kRows, D) | ptx::kIdescMnMajorB;
      const uint64_t q_desc = ptx::umma_desc_k_sw128(smem_base), k_desc = ptx::umma_desc_k_sw128(ring_base);
      const uint64_t v_desc = ptx::umma_desc_mn_sw128(ring_base, kHalfBytes);
      const bool one = ptx::elect_one();
      bool ok = true;
      const auto scores = [&](int t, int at) {
        const uint64_t q = q_desc + t * (kTileBytes >> 4), keys = k_desc + at * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          ptx::umma_f16_ss_by(one && ok, t * kRows, q + off, keys + off, idesc_s, k > 0);
        }
        ptx::umma_commit_by(one && ok, ptx::smem_u32(s_bar + t));
      };
      int stage = 1;
      uint32_t phase = 0;
      if (steps > 0)
        ok = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(q_bar), 0, abort_flag) &&
                           ptx::mbar_wait(ptx::smem_u32(full_bar), 0, abort_flag));
      ptx::tc_fence_after_sync();
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (tiles[t] > 0 && skip[t] == 0) scores(t, 0);
      ptx::umma_commit_by(one && ok, ptx::smem_u32(free_bar));
      for (int s = 0; s < steps; ++s) {
        const int v_stage = stage, k_stage = stage + 1 == kStages ? 0 : stage + 1;
        const uint32_t v_phase = phase, k_phase = k_stage == 0 ? phase ^ 1u : phase;
        const bool more = s + 1 < steps;
        const uint64_t values = v_desc + v_stage * (kTileBytes >> 4);
        if (ok)
          ok = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(full_bar + v_stage), v_phase, abort_flag) &&
                             (!more || ptx::mbar_wait(ptx::smem_u32(full_bar + k_stage), k_phase, abort_flag)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (s >= skip[t]) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (ok) ok = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(p_bar + 2 * t + c), (s - skip[t]) & 1, abort_flag));
              ptx::tc_fence_after_sync();
#pragma unroll
              for (int i = 0; i < kRows / 32; ++i) {
                const int k = c * (kRows / 32) + i;
                ptx::umma_f16_ts_by(one && ok, kColO + t * kRows, t * kRows + 8 * k, values + k * (2048 >> 4), idesc_o,
                                    s > skip[t] || k > 0);
              }
            }
          }
          if (more && s + 1 >= skip[t]) scores(t, k_stage);
        }
        ptx::umma_commit_by(one && ok, more ? ptx::smem_u32(free_bar + ((s + 1) & 3)) : ptx::smem_u32(o_bar));
        for (int x = 0; x < 2; ++x)
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
      }
    } else if (warp >= 8) {
      ptx::lower_registers<kOtherRegs>();
    } else {
      ptx::raise_registers<kSoftmaxRegs>();
      // ---------------------------------------------------------------- softmax
      const int t = warp >> 2, row = (warp & 3) * 32 + lane;
      const int query = it.first + t * p.tile_tokens + row / p.group;
      const bool real = row < p.tile_tokens * p.group && query < it.n;
      const int limit = real ? seen(query) : 0;
      const int first_limit = seen(it.first + t * p.tile_tokens);     // the fewest keys of a row
      const uint32_t lanes = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      const uint32_t col_s = lanes + t * kRows, col_o = lanes + kColO + t * kRows;
      bool alive = true;
      if (warp == 4 && tail) {
        // Behind the last key the last V tile holds another sequence's rows or whatever the page did; 0 * NaN is NaN.
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(tail_bar), 0, abort_flag));
        const int from = it.m - (steps - 1) * kRows;
        for (int e = lane; e < (kRows - from) * (D / 8); e += 32) {
          const int r = from + e / (D / 8), c = e % (D / 8);
          *reinterpret_cast<uint4*>(ring + kTileBytes + (c >> 3) * kHalfBytes + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && alive) ptx::mbar_arrive(ptx::smem_u32(full_bar + 1));
      }
      float top = -INFINITY, sum = 0.f;
      for (int s = skip[t]; s < steps; ++s) {
        const int turn = s - skip[t];
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(s_bar + t), turn & 1, abort_flag));
        if (!alive) break;
        ptx::tc_fence_after_sync();
        float x[kRows];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          ptx::tmem_ld_32x32b_x32(col_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
        ptx::tmem_ld_wait();
        const int begin = (steps - 1 - s) * kRows;
        if (begin + kRows > first_limit) {
#pragma unroll
          for (int c = 0; c < kRows; ++c)
            if (begin + c >= limit) x[c] = -INFINITY;
        }
        float most[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c + 8 <= kRows; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) most[i] = max3(most[i], x[c + 2 * i], x[c + 2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], x[kRows - 4 + i]);
        const float next = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2;
        if (turn == 0) {
          top = next;
        } else if (__any_sync(~0u, next > top + kLazy)) {
          const float raised = fmaxf(next, top);
          const float f = raised == top ? 1.f : exp2_approx(top - raised);
          top = raised;
          sum *= f;
          // (the scores were issued behind the last product into O, so that is done as well)
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld_32x32b_x32(col_o + 32 * c, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st_32x32b_x32(col_o + 32 * c, o);
          }
        }
        const float base = top == -INFINITY ? 0.f : top;
        // The exponential unit gives 16 results a cycle for the SM; every fourth pair goes through the multipliers instead.
        const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), base2 = pair(-base, -base);
        uint64_t part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint64_t arg = fma2(pair(x[64 * c + 2 * i], x[64 * c + 2 * i + 1]), scale2, base2);
            float2 e;
            if (i % 4 == 3) {
              e = exp2_poly(arg);
            } else {
              e = unpair(arg);
              e = make_float2(exp2_approx(e.x), exp2_approx(e.y));
            }
            part[i & 1] = add2(part[i & 1], pair(e.x, e.y));
            w[i] = pack16<T>(e.x, e.y);
          }
          ptx::tmem_st_32x32b_x32(col_s + 32 * c, w);
          // the product of this half may begin
          ptx::tmem_st_wait();
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(p_bar + 2 * t + c));
        }
        const float2 both = unpair(add2(part[0], part[1]));
        sum += both.x + both.y;
      }
      const int head = kv * p.group + row % p.group;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) +
                                            (static_cast<int64_t>(it.row0 + query) * p.heads + head) * p.dim);
      const bool any = tiles[t] > 0;
      if (any && alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(o_bar), 0, abort_flag));
      ptx::tc_fence_after_sync();
      const float inv = limit > 0 ? 1.f / sum : 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (any && alive) {
          ptx::tmem_ld_32x32b_x32(col_o + 32 * c, o);
          ptx::tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = limit > 0 ? pack16<T>(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv) : 0u;
          if (real && alive && 32 * c + 8 * i < p.dim) out[4 * c + i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && *abort_flag != 0) atomicCAS(p.status, 0, 0x900 | (static_cast<int>(blockIdx.x) << 12));
}

template <typename T, int D>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PrefillParams& p, cudaStream_t stream) {
  constexpr int smem = smem_bytes<D>();
  static_assert(smem <= 227 * 1024 && 2 * smem > kSmSharedBytes, "one CTA an SM: it takes all tensor memory");
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  auto kern = attn_prefill_kernel<T, D>;
  cudaError_t e = cudaSuccess;
  if (dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) attr_set[dev] = true;
  }
  // at most one item of each sequence is not full
  const int per_item = 2 * p.tile_tokens;
  const int64_t items = std::min<int64_t>(p.tokens, p.tokens / per_item + static_cast<int64_t>(p.sequences));
  if (items * p.kv_heads > 0x7fffffff) return B200Q_ERR_BAD_SHAPE;
  if (e == cudaSuccess)
    e = launch_overlapped(MAX_SHARED, kern, dim3(static_cast<unsigned>(items * p.kv_heads)), dim3(kThreads), smem, stream, tq,
                          tk, tv, p);
  if (e != cudaSuccess) {
    note_cuda_error(e);
    return B200Q_ERR_LAUNCH;
  }
  count_launch();
  return B200Q_OK;
}

}  // namespace

size_t attn_prefill_workspace(const b200q_attention&) { return 0; }

int launch_attn_prefill(const b200q_attention& a, void*, int* status, cudaStream_t stream) {
  PrefillParams p{};
  p.out = a.out;
  p.cu_q = a.cu_q, p.cu_k = a.cu_k, p.tables = a.tables, p.table_stride = a.table_stride;
  p.tokens = a.tokens, p.key_tokens = a.key_tokens, p.sequences = a.sequences;
  p.heads = a.heads, p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.dim = a.dim;
  p.pages = a.pages, p.page_size = a.page_size, p.table_width = a.table_width;
  p.tile_tokens = kRows / p.group;
  p.box_rows = kRows;
  while (a.page_size % p.box_rows != 0) p.box_rows /= 2;
  p.causal = a.causal;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = status;
  CUtensorMap tq, tk, tv;
  // queries: [tokens][key heads][group][dim]
  const uint64_t size[4] = {static_cast<uint64_t>(a.dim), static_cast<uint64_t>(p.group), static_cast<uint64_t>(a.kv_heads),
                            static_cast<uint64_t>(a.tokens)};
  int64_t stride[3] = {a.q.head, a.q.head * p.group, a.q.token};
  for (int i = 0; i < 3; ++i)
    if (size[i + 1] == 1) stride[i] = (a.dim + 7) / 8 * 8;      // says nothing, but has to be valid
  const uint32_t box[4] = {64, static_cast<uint32_t>(p.group), 1, static_cast<uint32_t>(p.tile_tokens)};
  if (!make_tensor_map_16(a.q.data, 4, size, stride, box, &tq) || !make_key_map(a.k, a, p.box_rows, &tk) ||
      !make_key_map(a.v, a, p.box_rows, &tv))
    return B200Q_ERR_LAUNCH;
  const bool bf = a.dtype == B200Q_DTYPE_BF16;
  if (a.dim <= 64)
    return bf ? launch<__nv_bfloat16, 64>(tq, tk, tv, p, stream) : launch<__half, 64>(tq, tk, tv, p, stream);
  return bf ? launch<__nv_bfloat16, 128>(tq, tk, tv, p, stream) : launch<__half, 128>(tq, tk, tv, p, stream);
}

}  // namespace b200q
