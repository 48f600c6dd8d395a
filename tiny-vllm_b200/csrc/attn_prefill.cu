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
// Keys go from the last tile, where the mask is, to the first.  `top` is the maximum of a row's first step.  Later steps do not
// look for theirs: as long as the sum of their weights stays small, `top` may stay as well; else it is raised, and O_t
// rescaled in place.  Weights reach 2^12 at most, rounded with the same relative error.
//
// Work: an item is two tiles of queries and their keys.  Where there are more items than SMs, or one of them might be long, a
// small kernel (attn_plan_kernel) lists them first, those with the most keys at the front, and CTAs, one an SM, take one
// after another; the next item's Q and K arrive under the last exponentials of the one before, whose output stands behind the
// first exponentials of the next.  An item with more than one and a half times an SM's share of all keys is cut into
// pieces, which leave fp32 partial results for a third kernel to join in their order: few queries over a long cached prefix
// then use the whole GPU.
//
// Rows whose scores are far from zero, and those beside a hidden value that is not finite, are taken once more by row_by_row.
//
// 8192 tokens, 32 query and 8 key heads of 128, causal: 430 us in short runs (1280 TFLOP/s), 495 back to back under the power cap.  A
// tile's step takes 3000 cycles for the 2048 of its and the other tile's products: 2000 of softmax, in which a warp alone on
// its quarter of the SM waits for instructions, then 1000 until the next scores are there, the tensor cores busy with the
// other tile for half of it.
//
// Warps: 0-3 and 4-7 softmax of tile 0 and 1, a row a thread; 8 issues the products; 9 brings Q, K and V; 10 fetches
// items; 11 clears the end of a sequence's last V tile.
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
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "registers");
constexpr int kCtrlBytes = 1024;
constexpr int kTmemCols = 512;
constexpr uint32_t kColO = 256;
constexpr float kMost = 4096.f, kMostLog2 = 12.f;  // the largest weight
constexpr float kFar = 1048576.f;                 // rows with larger maxima go to row_by_row
constexpr int kMinChunk = 8;                      // tiles of keys: the shortest piece that an item is cut into
constexpr int kFirstGroups = 6;                   // of 16 keys, whose weights are announced first
constexpr int kChecked = 48;                      // pairs of weights whose sum says whether the maximum follows
constexpr int kReaders = 11;                      // warps that read an item
constexpr int kItems = 4;                         // places for items that are on their way or worked on
constexpr int kSignals = 8;                       // more than the products can be ahead of the copies: stages / 2 + 1

template <int D>
constexpr int stages() { return D == 128 ? 5 : 10; }
template <int D>
constexpr int smem_bytes() { return (2 + stages<D>()) * kRows * D * 2 + kCtrlBytes; }

// The queries of one sequence that a CTA works on, and the part of the sequence's keys.
struct alignas(16) Item {
  int b, n, m;          // sequence, its queries and keys; b < 0: no more items
  int first;            // first query of the item in its sequence
  int row0, key0;       // where the sequence begins in q and in packed keys
  int lo, hi;           // tiles of keys
  int slot, pieces;     // pieces > 1: place of this piece's partial results (times key heads)
  int kv, pad;
  struct {
    int skip;           // steps that a tile of rows sits out at the beginning; all of them where it has no rows or sees no key
    int cols;           // how many keys of its first step's tile it sees
  } part[2];
};
struct Header {
  int units, next, joins, pad;
};

struct PrefillParams {
  b200q_view q, k, v;   // for row_by_row
  void* out;
  const int32_t *cu_q, *cu_k, *tables;
  int64_t table_stride;
  int tokens, key_tokens, sequences, heads, kv_heads, group, dim, pages, page_size, table_width;
  int tile_tokens;      // queries of a tile: 128 / group
  int group_inverse;    // row / group = row * group_inverse >> 16
  int box_rows;
  int causal;
  float scale_log2;
  int split, sms, ctas, most_units;
  Header* header;       // NULL: a CTA for each item, no list
  Item* units;          // the list; kv and part are not set, nor in `joins` lo and hi
  Item* joins;          // items that were cut: slot of their first piece
  float* part_o;        // [slot][key head][2 tiles x 128 rows][D]
  float2* part_ml;      // maximum, sum
  int* status;
};

__device__ __forceinline__ int queries_of(const PrefillParams& p, int from, int to) {
  return max(min(to, p.tokens) - min(max(from, 0), p.tokens), 0);
}
__device__ __forceinline__ int items_of(const PrefillParams& p, int n) {
  return (n + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
}
// Keys that query i sees: [0, seen).
__device__ __forceinline__ int seen_by(const PrefillParams& p, const Item& it, int i) {
  return max(0, p.causal ? min(it.m, it.m - it.n + i + 1) : it.m);
}
__device__ __forceinline__ Item sequence_of(const PrefillParams& p, const int* cu_q, const int* cu_k, int b) {
  Item it{};
  it.b = b, it.n = queries_of(p, cu_q[b], cu_q[b + 1]), it.row0 = min(max(cu_q[b], 0), p.tokens);
  it.key0 = cu_k[b], it.pieces = 1;
  int64_t m = cu_k[b + 1] - static_cast<int64_t>(it.key0);
  if (p.page_size > 0) m = min(m, static_cast<int64_t>(p.table_width) * p.page_size);
  else m = it.key0 < 0 ? 0 : min(m, static_cast<int64_t>(p.key_tokens) - it.key0);
  it.m = static_cast<int>(min(max(m, int64_t{0}), static_cast<int64_t>(INT_MAX - kRows)));
  return it;
}
__device__ __forceinline__ void set_item(const PrefillParams& p, Item& it, int index) {
  it.first = index * 2 * p.tile_tokens;
  it.lo = 0;
  it.hi = (seen_by(p, it, min(it.first + 2 * p.tile_tokens, it.n) - 1) + kRows - 1) / kRows;
}

// Lists the items by falling number of keys.  One block: a warp takes a sequence, a lane an item.
constexpr int kPlanThreads = 1024, kBuckets = 1024, kPlanCached = 2048;
__global__ void __launch_bounds__(kPlanThreads) attn_plan_kernel(const PrefillParams p) {
  __shared__ int count[kBuckets], sums[32], slots, joins, cached[2][kPlanCached];
  __shared__ unsigned long long work;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  count[threadIdx.x] = 0;
  if (threadIdx.x == 0) slots = joins = 0, work = 0;
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  // the lengths are read three times
  const int *cu_q = p.cu_q, *cu_k = p.cu_k;
  if (p.sequences < kPlanCached) {
    for (int b = threadIdx.x; b <= p.sequences; b += kPlanThreads) cached[0][b] = cu_q[b], cached[1][b] = cu_k[b];
    cu_q = cached[0], cu_k = cached[1];
  }
  __syncthreads();
  unsigned long long mine = 0;
  for (int b = p.split ? warp : p.sequences; b < p.sequences; b += 32) {
    Item it = sequence_of(p, cu_q, cu_k, b);
#pragma unroll 1
    for (int i = lane; i < items_of(p, it.n); i += 32) {
      set_item(p, it, i);
      mine += it.hi;
    }
  }
  if (mine > 0) atomicAdd(&work, mine);
  __syncthreads();
  // Items with more than one and a half times an SM's share are cut into shares: a cut costs the writing and reading of
  // fp32 sums (8 x 128 queries over 2000 keys, 17 tiles at a share of 15: cut 75 us, whole 57).
  int chunk = INT_MAX;
  if (p.split)
    chunk = max(static_cast<int>(min(static_cast<float>(work) * p.kv_heads / p.sms, 1e9f)) + 1, kMinChunk);
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int b = warp; b < p.sequences; b += 32) {
      Item it = sequence_of(p, cu_q, cu_k, b);
#pragma unroll 1
      for (int i = lane; i < items_of(p, it.n); i += 32) {
        set_item(p, it, i);
        const int all = it.hi;
        it.pieces = all > chunk && all - chunk > chunk / 2 ? (all + chunk - 1) / chunk : 1;
        const int each = it.pieces > 1 ? all / it.pieces : all, rest = all - each * it.pieces;
        if (pass == 1 && it.pieces > 1) {
          it.slot = atomicAdd(&slots, it.pieces);
          p.joins[atomicAdd(&joins, 1)] = it;
        }
#pragma unroll 1
        for (int c = 0; c < it.pieces; ++c) {
          it.lo = c * each + min(c, rest);
          it.hi = it.lo + each + (c < rest);
          const int at = atomicAdd(&count[kBuckets - 1 - min(it.hi - it.lo, kBuckets - 1)], 1);
          if (pass == 1) {
            if (at < p.most_units) p.units[at] = it;
            ++it.slot;
          }
        }
      }
    }
    __syncthreads();
    if (pass == 0) {      // where each bucket begins
      const int own = count[threadIdx.x];
      int upto = own;
      for (int x = 1; x < 32; x *= 2) {
        const int o = __shfl_up_sync(~0u, upto, x);
        if (lane >= x) upto += o;
      }
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      if (warp == 0) {
        int before = sums[lane];
        for (int x = 1; x < 32; x *= 2) {
          const int o = __shfl_up_sync(~0u, before, x);
          if (lane >= x) before += o;
        }
        sums[lane] = before;
      }
      __syncthreads();
      if (warp > 0) upto += sums[warp - 1];
      count[threadIdx.x] = upto - own;
      if (threadIdx.x == kPlanThreads - 1) {
        // more than sequences that follow one another can have: the list ends where its memory does
        if (upto > p.most_units) atomicCAS(p.status, 0, 0xa03);
        p.header->units = min(upto, p.most_units), p.header->next = p.ctas;
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) p.header->joins = joins;
}

// Where key `pos` of an item stands in x; -1: in a page outside of the cache, which counts as zeros, or behind the last key.
__device__ __forceinline__ int64_t place_of(const PrefillParams& p, const Item& it, const b200q_view& x, int pos) {
  if (pos >= it.m) return -1;
  if (p.page_size == 0) return static_cast<int64_t>(it.key0 + pos) * x.token + it.kv * x.head;
  const int page = p.tables[it.b * p.table_stride + pos / p.page_size];
  return page < 0 || page >= p.pages ? -1 : page * x.page + pos % p.page_size * x.token + it.kv * x.head;
}

// A warp's 32 rows of tile t of an item (or of a piece of it) once more, the result written over the former one: where a maximum is
// far from zero (odd = 2), or where sums are not finite though the weights are (1) and a value that is not finite stands behind what a
// row sees (its weight is 0, and 0 * inf is NaN).  Exponents are scale (x - max x), weights stay in fp32, and only what a row sees
// is multiplied.  Scores by mma.sync, 16 rows x 8 keys at a time, straight from memory.  Rare, so it may be slow: 8192 tokens of
// 32 / 8 heads of 128 whose scores are all far take 49 ms, 2700 cycles for each of an item's keys (beyond 700,000 of them the
// other warps' waits run out, and the call ends with a device status).  A function of its own: the same work between the other
// steps cost these up to 9 %.
template <typename T, int D>
__device__ __noinline__ void row_by_row(const PrefillParams& p, const Item& it, int t, int my_row, int odd) {
  const int lane = threadIdx.x & 31, gid = lane >> 2, tid = lane & 3, row0 = my_row - lane;
  const auto limit_of = [&](int row) {      // keys of the piece that a row sees; -1: no row
    const int of = row / p.group, query = it.first + t * p.tile_tokens + of;
    return of < p.tile_tokens && query < it.n ? min(seen_by(p, it, query), it.hi * kRows) : -1;
  };
  if (!__any_sync(~0u, odd == 2)) {
    // is there a value at all that is not finite, behind the fewest keys that a row sees?
    const int mine = limit_of(row0 + lane), pieces = p.dim / 8, fewest = __reduce_min_sync(~0u, mine < 0 ? INT_MAX : mine);
    const int from = max(fewest, it.lo * kRows), keys = min(it.m, (it.hi - it.part[t].skip) * kRows) - from;
    float zero = 0.f;
#pragma unroll 1
    for (int e0 = 0; e0 < keys * pieces; e0 += 32) {
      const int e = min(e0 + lane, keys * pieces - 1);
      const int64_t at = place_of(p, it, p.v, from + e / pieces);
      float x[8];
      unpack8<T>(static_cast<const T*>(p.v.data) + (at < 0 ? 0 : at) + e % pieces * 8, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) zero = at < 0 ? zero : fmaf(x[i], 0.f, zero);
    }
    if (!__any_sync(~0u, zero != 0.f)) return;      // (NaN, too, is not 0)
  }
  __syncwarp();      // the former result was written by other lanes
#pragma unroll 1
  for (int block = 0; block < 32; block += 16) {
    int row[2], limit[2];
    float most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, o[D / 8][4];
    const T* q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[h] = row0 + block + gid + 8 * h, limit[h] = limit_of(row[h]);
      const int query = it.row0 + it.first + t * p.tile_tokens + row[h] / p.group, head = it.kv * p.group + row[h] % p.group;
      q[h] = static_cast<const T*>(p.q.data) + (limit[h] < 0 ? 0 : query * p.q.token + head * p.q.head);
    }
    uint32_t a[D / 16][4];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * k + 8 * (i >> 1) + 2 * tid;
        a[k][i] = limit[i & 1] >= 0 && d < p.dim ? *reinterpret_cast<const uint32_t*>(q[i & 1] + d) : 0u;
      }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    const int all = __reduce_max_sync(~0u, max(limit[0], limit[1]));
#pragma unroll 1
    for (int j = it.lo * kRows; j < all; j += 8) {
      const int64_t k_at = place_of(p, it, p.k, j + gid), v_at = place_of(p, it, p.v, j + gid);      // of the key that a lane has in a product
      const T* key = static_cast<const T*>(p.k.data) + (k_at < 0 ? 0 : k_at);
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = 16 * k + 8 * i + 2 * tid;
          b[i] = k_at >= 0 && d < p.dim ? *reinterpret_cast<const uint32_t*>(key + d) : 0u;
        }
        mma_16<T>(s, a[k][0], a[k][1], a[k][2], a[k][3], b[0], b[1]);
      }
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {      // keys 2 tid and 2 tid + 1 of rows gid, gid + 8
        float to = most[h];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (j + 2 * tid + i >= limit[h]) s[2 * h + i] = -INFINITY;
          to = fmaxf(to, s[2 * h + i]);
        }
        to = fmaxf(to, __shfl_xor_sync(~0u, to, 1));
        to = fmaxf(to, __shfl_xor_sync(~0u, to, 2));
        f[h] = to == most[h] ? 1.f : exp2_approx((most[h] - to) * p.scale_log2);
        most[h] = to;
        const float base = to == -INFINITY ? 0.f : to;
        sum[h] *= f[h];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[2 * h + i] = exp2_approx((s[2 * h + i] - base) * p.scale_log2);
          sum[h] += s[2 * h + i];
        }
      }
      if (__any_sync(~0u, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
      }
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const int from = (lane & 28) | (i >> 1);
        const float w0 = __shfl_sync(~0u, i & 1 ? s[1] : s[0], from), w1 = __shfl_sync(~0u, i & 1 ? s[3] : s[2], from);
        const int64_t at = __shfl_sync(~0u, v_at, 4 * i);
        const T* value = static_cast<const T*>(p.v.data) + at + 2 * tid;
        if (at < 0) continue;
        const bool sees0 = j + i < limit[0], sees1 = j + i < limit[1];
        uint32_t v[D / 8];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) v[n] = 8 * n + 2 * tid < p.dim ? *reinterpret_cast<const uint32_t*>(value + 8 * n) : 0u;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          const float x = static_cast<float>(reinterpret_cast<const T*>(&v[n])[0]), y = static_cast<float>(reinterpret_cast<const T*>(&v[n])[1]);
          if (sees0) o[n][0] = fmaf(w0, x, o[n][0]), o[n][1] = fmaf(w0, y, o[n][1]);
          if (sees1) o[n][2] = fmaf(w1, x, o[n][2]), o[n][3] = fmaf(w1, y, o[n][3]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(~0u, sum[h], 1);
      sum[h] += __shfl_xor_sync(~0u, sum[h], 2);
      if (limit[h] < 0) continue;
      if (it.pieces > 1) {
        const int64_t at = (static_cast<int64_t>(it.slot) * p.kv_heads + it.kv) * 2 * kRows + t * kRows + row[h];
        if (tid == 0) p.part_ml[at] = make_float2(most[h] * p.scale_log2, sum[h]);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(p.part_o + at * D + 8 * n + 2 * tid) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
      } else {
        const float inv = inverse(sum[h]);
        const int query = it.row0 + it.first + t * p.tile_tokens + row[h] / p.group, head = it.kv * p.group + row[h] % p.group;
        T* to = static_cast<T*>(p.out) + (static_cast<int64_t>(query) * p.heads + head) * p.dim + 2 * tid;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          if (8 * n < p.dim) *reinterpret_cast<uint32_t*>(to + 8 * n) = pack16<T>(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
      }
    }
    __syncwarp();
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                    const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PrefillParams p) {
  constexpr int kHalves = D / 64;
  constexpr int kHalfBytes = kRows * 128;
  constexpr int kTileBytes = kRows * D * 2;
  constexpr int kStages = stages<D>();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + 2 * kTileBytes;
  uint8_t* ctrl = ring + kStages * kTileBytes;
  Item* items = reinterpret_cast<Item*>(ctrl);              // [items]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(items + kItems);   // [stages] a K or V tile is there
  uint64_t* free_bar = full_bar + kStages;                  // [signals], in turn: products up to a step are done
  uint64_t* s_bar = free_bar + kSignals;                           // [2] scores of a tile are there
  uint64_t* p_bar = s_bar + 2;                              // [2][2] its weights are, of the first keys and the others
  uint64_t* o_bar = p_bar + 4;                              // [2] all products of an item are done
  uint64_t* q_bar = o_bar + 2;
  uint64_t* tail_bar = q_bar + 1;                           // [stages] a last V tile, before its end is cleared
  uint64_t* want_bar = tail_bar + kStages;                  // the next item is wanted
  uint64_t* item_bar = want_bar + 1;                        // [items] an item is there
  uint64_t* read_bar = item_bar + kItems;                   // [items] all have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(read_bar + kItems);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert(kItems * sizeof(Item) + 8 * (2 * kStages + kSignals + 10 + 2 * kItems) + 8 <= kCtrlBytes, "control words");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = ptx::smem_u32(smem), ring_base = smem_base + 2 * kTileBytes;
  if ((smem_base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 0x200);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(ptx::smem_u32(full_bar + s), 1);
    for (int e = 0; e < kSignals; ++e) ptx::mbar_init(ptx::smem_u32(free_bar + e), 1);
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(s_bar + t), 1);
      ptx::mbar_init(ptx::smem_u32(p_bar + 2 * t), 4);
      ptx::mbar_init(ptx::smem_u32(p_bar + 2 * t + 1), 4);
      ptx::mbar_init(ptx::smem_u32(o_bar + t), 1);
    }
    for (int k = 0; k < kItems; ++k) {
      ptx::mbar_init(ptx::smem_u32(item_bar + k), 1);
      ptx::mbar_init(ptx::smem_u32(read_bar + k), kReaders);
    }
    ptx::mbar_init(ptx::smem_u32(q_bar), 1);
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(ptx::smem_u32(tail_bar + s), 1);
    ptx::mbar_init(ptx::smem_u32(want_bar), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::tma_prefetch_desc(&tmap_q);
    ptx::tma_prefetch_desc(&tmap_k);
    ptx::tma_prefetch_desc(&tmap_v);
  }
  if (warp == 8) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const uint32_t tmem_base = *tmem_slot;      // all columns: 0, which the products' constants rely on
  if (tmem_base != 0 && threadIdx.x == 0) {
    atomicCAS(p.status, 0, 0x200);
    *abort_flag = 1;
  }

  bool alive = true;
  int turn = 0;
  const auto fetch = [&](Item& it) -> bool {
    const int slot = turn % kItems;
    if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(item_bar + slot), (turn / kItems) & 1, abort_flag));
    it = items[slot];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(read_bar + slot));
    ++turn;
    return alive && it.b >= 0;
  };
  if (warp == 10) {
    ptx::lower_registers<kOtherRegs>();
    // ---------------------------------------------------------------- items
    for (int k = 0;; ++k) {
      Item it{};
      it.b = -1;
      // The next one is taken when the copies of the one before are on their way: taken earlier, it might be left waiting
      // while another CTA has nothing to do.
      if (k > 0 && alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(want_bar), (k - 1) & 1, abort_flag));
      if (p.header != nullptr) {
        int at = static_cast<int>(blockIdx.x);
        if (k > 0) at = __shfl_sync(~0u, lane == 0 ? atomicAdd(&p.header->next, 1) : 0, 0);
        const int unit = at / p.kv_heads;
        if (unit < p.most_units) {      // (both loads at once)
          it = p.units[unit];
          it.kv = at - unit * p.kv_heads;
          if (unit >= *const_cast<const volatile int*>(&p.header->units)) {      // nothing was written there
            it = Item{};
            it.b = -1;
          }
        }
      } else if (k == 0) {
        // the blockIdx.x / kv_heads-th item of all sequences
        int before = static_cast<int>(blockIdx.x) / p.kv_heads;
        for (int b0 = 0; b0 < p.sequences; b0 += 32) {
          const int own = b0 + lane < p.sequences ? items_of(p, queries_of(p, p.cu_q[b0 + lane], p.cu_q[b0 + lane + 1])) : 0;
          int upto = own;
          for (int x = 1; x < 32; x *= 2) {
            const int o = __shfl_up_sync(~0u, upto, x);
            if (lane >= x) upto += o;
          }
          const uint32_t over = __ballot_sync(~0u, upto > before);
          if (over != 0) {
            const int l = __ffs(over) - 1;
            before -= __shfl_sync(~0u, upto - own, l);
            it = sequence_of(p, p.cu_q, p.cu_k, b0 + l);
            set_item(p, it, before);
            it.kv = static_cast<int>(blockIdx.x) % p.kv_heads;
            break;
          }
          before -= __shfl_sync(~0u, upto, 31);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int from = it.first + t * p.tile_tokens, to = min(from + p.tile_tokens, it.n);
        const int seen = from < to ? seen_by(p, it, to - 1) : 0, steps = it.hi - it.lo;
        it.part[t].skip = min(max(it.hi - (seen + kRows - 1) / kRows, 0), steps);
        it.part[t].cols = min(seen - (it.hi - 1 - it.part[t].skip) * kRows, kRows);
      }
      if (k >= kItems && alive)
        alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(read_bar + k % kItems), (k / kItems - 1) & 1, abort_flag));
      if (lane == 0 && alive) {
        items[k % kItems] = it;
        ptx::mbar_arrive(ptx::smem_u32(item_bar + k % kItems));
      }
      if (it.b < 0 || !alive) break;
    }
  } else if (warp == 9) {
    ptx::lower_registers<kOtherRegs>();
    // ---------------------------------------------------------------- Q, K and V
    const int boxes = kRows / p.box_rows;
    int stage = 0, freed = 0, signal = 0, q_free = -1;
    int holder = -1;      // lane l: the signal that frees place l of the ring
    uint32_t phase = 0, tails = 0, tail_phase = 0, queries = 0;      // tails, tail_phase: a bit for each place of the ring
    const auto wait_for = [&](int event) {
      for (; freed <= event; ++freed)
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(free_bar + (freed & (kSignals - 1))), (freed / kSignals) & 1, abort_flag));
    };
    Item it;
    while (fetch(it)) {
      const int steps = it.hi - it.lo;
      if (steps == 0) {
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(want_bar));
        continue;
      }
      const bool any[2] = {it.part[0].skip < steps, it.part[1].skip < steps}, tail = it.hi * kRows > it.m;
      wait_for(q_free);      // the scores of the item before are done
      if (lane == 0 && alive) {
        const uint32_t bar = ptx::smem_u32(q_bar);
        ptx::mbar_arrive_expect_tx(bar, p.tile_tokens * p.group * 128 * kHalves * (any[0] + any[1]));
#pragma unroll
        for (int t = 0; t < 2; ++t)
          for (int h = 0; h < kHalves && any[t]; ++h)
            ptx::tma_load_4d(smem_base + t * kTileBytes + h * kHalfBytes, &tmap_q, bar, h * 64, 0, it.kv,
                             it.row0 + it.first + t * p.tile_tokens);
      }
      __syncwarp();
      ++queries;
      const int32_t* table = p.page_size > 0 ? p.tables + it.b * p.table_stride : nullptr;
      int page = 0;
      for (int s = 0; s < steps; ++s) {
        const int begin = (it.hi - 1 - s) * kRows;
        int at = it.key0 + begin, held = 1, mine = 0;
        if (p.page_size > 0) {
          // pages of the next 32 boxes at a time, from the last key backwards
          if (s * boxes % 32 == 0) {
            const int64_t pos = static_cast<int64_t>(it.hi) * kRows - static_cast<int64_t>(s * boxes + lane + 1) * p.box_rows;
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
          wait_for(__shfl_sync(~0u, holder, stage));
          const bool last_values = x == 1 && s == 0 && tail;
          const uint32_t bar = ptx::smem_u32((last_values ? tail_bar : full_bar) + stage);
          if (lane == 0 && alive) ptx::mbar_arrive_expect_tx(bar, held * p.box_rows * D * 2);
          __syncwarp();
          if (lane < held && alive)
            for (int h = 0; h < kHalves; ++h)
              ptx::tma_load_4d(ring_base + stage * kTileBytes + h * kHalfBytes + lane * p.box_rows * 128,
                               x == 0 ? &tmap_k : &tmap_v, bar, h * 64, it.kv, at, mine);
          if (last_values) {
            tail_phase ^= (tails >> stage & 1u) << stage;      // of the last copy
            tails |= 1u << stage;
          }
          // signals of an item: the first scores; then each step's values together with the next one's scores
          if (lane == stage) holder = signal + s + x;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(want_bar));
      q_free = signal + steps - 1;
      signal += steps + 1;
    }
    wait_for(signal - 1);      // no signal is on its way to a barrier of a CTA that has ended
    __syncwarp();
    if (lane == 0) {
      if (*abort_flag != 0) ptx::drain_ring(full_bar, kStages, stage, phase);
      for (int s = 0; s < kStages; ++s)
        if (*abort_flag != 0 && (tails >> s & 1u) != 0u) ptx::drain_ring(tail_bar + s, 1, 1, tail_phase >> s & 1u);
      if (*abort_flag != 0 && queries > 0) ptx::drain_ring(q_bar, 1, 1, (queries - 1) & 1);
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
    const auto scores = [&](int t, int at, uint32_t idesc) {
      const uint64_t q = q_desc + t * (kTileBytes >> 4), keys = k_desc + at * (kTileBytes >> 4);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
        ptx::umma_f16_ss_by(one && alive, t * kRows, q + off, keys + off, idesc, k > 0);
      }
      ptx::umma_commit_by(one && alive, ptx::smem_u32(s_bar + t));
    };
    int stage = 0, signal = 0;
    uint32_t phase = 0, q_phase = 0, p_phase[2] = {0, 0};
    // the first tile of keys of a tile of rows counts up to the last one seen, in sixteens
    const auto groups_first = [&](const Item& it, int t) { return (it.part[t].cols + 15) >> 4; };
    const auto idesc_first = [&](const Item& it, int t) { return ptx::umma_idesc(1u, ab, kRows, groups_first(it, t) * 16); };
    const auto fetch_keys = [&](Item& it) -> bool {
      while (fetch(it))
        if (it.hi > it.lo) return true;
      return false;
    };
    Item it;
    while (fetch_keys(it)) {
      const int steps = it.hi - it.lo;
      if (alive)
        alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(q_bar), q_phase, abort_flag) &&
                              ptx::mbar_wait(ptx::smem_u32(full_bar + stage), phase, abort_flag));
      q_phase ^= 1u;
      ptx::tc_fence_after_sync();
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (it.part[t].skip == 0) scores(t, stage, idesc_first(it, t));
      ptx::umma_commit_by(one && alive, ptx::smem_u32(free_bar + (signal++ & (kSignals - 1))));
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
      for (int s = 0; s < steps; ++s) {
        const int v_stage = stage, k_stage = stage + 1 == kStages ? 0 : stage + 1;
        const uint32_t v_phase = phase, k_phase = k_stage == 0 ? phase ^ 1u : phase;
        const bool more = s + 1 < steps;
        const uint64_t values = v_desc + v_stage * (kTileBytes >> 4);
        if (alive)
          alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(full_bar + v_stage), v_phase, abort_flag) &&
                                (!more || ptx::mbar_wait(ptx::smem_u32(full_bar + k_stage), k_phase, abort_flag)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (s >= it.part[t].skip) {
            const int groups = s == it.part[t].skip ? groups_first(it, t) : kRows / 16;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(p_bar + 2 * t + c), p_phase[t], abort_flag));
              ptx::tc_fence_after_sync();
#pragma unroll
              for (int k = c * kFirstGroups; k < (c == 0 ? kFirstGroups : kRows / 16); ++k)
                ptx::umma_f16_ts_by(one && alive && k < groups, kColO + t * kRows, t * kRows + 8 * k, values + k * (2048 >> 4),
                                    idesc_o, s > it.part[t].skip || k > 0);
            }
            p_phase[t] ^= 1u;
            if (!more) ptx::umma_commit_by(one && alive, ptx::smem_u32(o_bar + t));
          }
          if (more && s + 1 >= it.part[t].skip)
            scores(t, k_stage, s + 1 == it.part[t].skip ? idesc_first(it, t) : idesc_s);
        }
        ptx::umma_commit_by(one && alive, ptx::smem_u32(free_bar + (signal++ & (kSignals - 1))));
        for (int x = 0; x < 1 + more; ++x)
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
      }
    }
  } else if (warp == 11) {
    ptx::lower_registers<kOtherRegs>();
    // ---------------------------------------------------------------- ends
    // Behind the last key the last V tile holds another sequence's rows or whatever the page did, and 0 * NaN is NaN: cleared
    // up to the next multiple of 16, which is what the products read.
    int stage = 0;
    uint32_t tail_phase = 0;      // a bit for each place of the ring: the next copy's
    Item it;
    while (fetch(it)) {
      const int steps = it.hi - it.lo;
      if (steps > 0 && it.hi * kRows > it.m) {
        const int place = stage + 1 == kStages ? 0 : stage + 1, from = it.m - (it.hi - 1) * kRows;
        // A barrier for each place: the next item's last values may be on their way before these are there.
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(tail_bar + place), tail_phase >> place & 1u, abort_flag));
        tail_phase ^= 1u << place;
        for (int e = lane; e < (((from + 15) & ~15) - from) * (D / 8); e += 32) {
          const int r = from + e / (D / 8), c = e % (D / 8);
          *reinterpret_cast<uint4*>(ring + place * kTileBytes + (c >> 3) * kHalfBytes + r * 128 + (c & 7) * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && alive) ptx::mbar_arrive(ptx::smem_u32(full_bar + place));
      }
      stage = (stage + 2 * steps) % kStages;
    }
  } else {
    ptx::raise_registers<kSoftmaxRegs>();
    // ---------------------------------------------------------------- softmax
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const int row_query = row * p.group_inverse >> 16;      // row / group
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t col_s = lanes + t * kRows, col_o = lanes + kColO + t * kRows;
    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
    uint32_t s_phase = 0, o_phase = 0;
    // A thread has its row's values one after another: it writes whole sectors of 32 bytes, where rows begin on such boundaries.  (By way
    // of shared memory, in whole lines, it took as long, and a place of the ring.)
    const auto write = [&](uint8_t* row, const uint32_t* v, int from, int bytes) {      // values `from` to from + 32 of a row
      if (((reinterpret_cast<uintptr_t>(row) | bytes) & 31u) == 0u) {
        if (from < bytes) ptx::st_global_32(row + from, v);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (from + 16 * i < bytes) *reinterpret_cast<uint4*>(row + from + 16 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    };
    // An item's result, where tile t has one; `any`: there are sums.  Returns what row_by_row has to know of the row: 0 where it is done.
    const auto output = [&](const Item& it, bool any, bool sees, float top, float sum) {
      const int to = it.first + t * p.tile_tokens;
      const bool real = row < min(it.n - to, p.tile_tokens) * p.group;
      uint64_t zero[4] = {0, 0, 0, 0};      // sums of 0 * o
      const auto odd = [&] {
        const float2 z = unpair(add2(add2(zero[0], zero[1]), add2(zero[2], zero[3])));
        return !real ? 0 : top == INFINITY ? 2 : sees && sum < INFINITY && !(z.x + z.y == 0.f) ? 1 : 0;
      };
      if (it.pieces > 1) {
        const int64_t at = (static_cast<int64_t>(it.slot) * p.kv_heads + it.kv) * 2 * kRows + t * kRows + row;
        if (real) p.part_ml[at] = make_float2(top, sum);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          if (!any) break;
          uint32_t o[32];
          ptx::tmem_ld_32x32b_x32(col_o + 32 * c, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) zero[i & 3] = fma2(pair(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), pair(0.f, 0.f), zero[i & 3]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (real) write(reinterpret_cast<uint8_t*>(p.part_o + at * D), o + 8 * i, c * 128 + 32 * i, D * 4);
        }
        return odd();
      }
      // rows of one query are neighbours; the next query is all heads further
      uint8_t* to_row = reinterpret_cast<uint8_t*>(
          static_cast<T*>(p.out) + (static_cast<int64_t>(it.row0 + to + row_query) * p.heads + it.kv * p.group + row - row_query * p.group) * p.dim);
      const float inv = inverse(sum);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32], v[16];
        if (any) {
          ptx::tmem_ld_32x32b_x32(col_o + 32 * c, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) zero[i & 3] = fma2(pair(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), pair(0.f, 0.f), zero[i & 3]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 r = unpair(mul2(pair(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), pair(inv, inv)));
          v[i] = sees ? pack16<T>(r.x, r.y) : 0u;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (real) write(to_row, v + 8 * i, c * 64 + 32 * i, p.dim * 2);
      }
      return odd();
    };
    uint32_t x[kRows], e16[kRows / 2];
    uint64_t part[2];
    float top = 0.f, most[4];
    // An exponent is scale x - top, with top = scale max x rounded: an error of a factor that a row's weights share, 2^(2^-4) where top is
    // kFar, but without bounds beyond.  Such a row is marked by an infinite maximum, its weights come out as 0, and row_by_row
    // takes it once more behind the output.
    const auto marked = [&](float x) { return fabsf(x) > kFar && x != -INFINITY ? INFINITY : x; };
    // Weights of pairs [from, to), eight at a time; sums, conversions and maxima (of the scores behind kChecked) of eight
    // stand beside the exponentials of the next.  The exponential unit gives 16 results a cycle for the SM; every eighth pair
    // goes through the multipliers instead (8 x 1024 tokens: every 4th 96 us, every 8th 93).
    const auto weights = [&](int from, int to) {
      const float base = top == -INFINITY ? 0.f : -top;
      const uint64_t base2 = pair(base, base);
      float2 e[2][8];
#pragma unroll
      for (int b = from / 8; b <= to / 8; ++b) {
        if (b < to / 8) {
          uint64_t arg[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            arg[i] = fma2(pair(__uint_as_float(x[16 * b + 2 * i]), __uint_as_float(x[16 * b + 2 * i + 1])), scale2, base2);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i % 8 == 7) {
              e[b & 1][i] = exp2_poly(arg[i]);
            } else {
              const float2 v = unpair(arg[i]);
              e[b & 1][i] = make_float2(exp2_approx(v.x), exp2_approx(v.y));
            }
          }
        }
        if (b > from / 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = 8 * (b - 1) + i;
            const float2 v = e[(b - 1) & 1][i];
            part[i & 1] = add2(part[i & 1], pair(v.x, v.y));
            e16[at] = pack16<T>(v.x, v.y);
            // (the maximum of the scores whose weights a sum does not check: those behind kChecked and, as exp2_poly is not
            // for arguments above 127, its own)
            if (at < kChecked && at % 3 == 0) {
              const int c = 2 * kChecked + 2 * (at / 3);
              most[i & 3] = max3(most[i & 3], __uint_as_float(x[c]), __uint_as_float(x[c + 1]));
            }
            if (at < kChecked && i % 8 == 7) most[i & 3] = max3(most[i & 3], __uint_as_float(x[2 * at]), __uint_as_float(x[2 * at + 1]));
          }
        }
      }
    };
    const auto announce = [&](int c) {      // the product of these weights may begin
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(p_bar + 2 * t + c));
    };
    const auto load = [&](int c) {      // columns 32 c on
      ptx::tmem_ld_32x32b_x32(col_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
    };
    // The item whose result is still in O: its place, and this row's statistics.
    int done = -1;
    bool done_any = false, done_sees = false;
    float done_top = 0.f, done_sum = 0.f;
    for (int k = 0;; ++k) {
      const int slot = k % kItems;
      const Item& it = items[slot];      // read where it is: it would take registers
      if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(item_bar + slot), (k / kItems) & 1, abort_flag));
      if (!alive) break;
      const bool end = it.b < 0;
      const int hi = it.hi, steps = end ? 0 : hi - it.lo, skip = it.part[t].skip, cols = it.part[t].cols;
      const bool any = !end && skip < steps;
      int limit = 0;                                                           // keys that the row sees
      {
        const int query = it.first + t * p.tile_tokens + row_query;
        if (!end && row_query < p.tile_tokens && query < it.n) limit = seen_by(p, it, query);
      }
      const int first_limit = seen_by(p, it, it.first + t * p.tile_tokens);     // the fewest keys of a row
      const auto mask = [&](int c, int begin) {      // columns 32 c on
        const int rel = limit - begin - 32 * c;
        const uint32_t sees = rel >= 32 ? ~0u : rel <= 0 ? 0u : (1u << rel) - 1u;
#pragma unroll
        for (int i = 0; i < 32; ++i) x[32 * c + i] = (sees >> i) & 1u ? x[32 * c + i] : __float_as_uint(-INFINITY);
      };
      float sum = 0.f;
      top = -INFINITY;
      if (any) {
        // ---- first step: the maximum comes first
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(s_bar + t), s_phase, abort_flag));
        if (!alive) break;
        s_phase ^= 1u;
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) load(c);
        ptx::tmem_ld_wait();
        const int begin = (hi - 1 - skip) * kRows;
        if (begin + kRows > first_limit) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask(c, begin);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = __uint_as_float(x[i]);
#pragma unroll
        for (int c = 4; c + 8 <= kRows; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) most[i] = max3(most[i], __uint_as_float(x[c + 2 * i]), __uint_as_float(x[c + 2 * i + 1]));
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], __uint_as_float(x[kRows - 4 + i]));
        top = marked(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2);
        part[0] = part[1] = pair(0.f, 0.f);
        weights(0, 32);
        ptx::tmem_st_32x32b_x32(col_s, *reinterpret_cast<uint32_t(*)[32]>(e16));
        if (cols > kRows / 2) {      // else no row sees the second half
          weights(32, 64);
          ptx::tmem_st_32x32b_x32(col_s + 32, *reinterpret_cast<uint32_t(*)[32]>(e16 + 32));
        }
        const float2 both = unpair(add2(part[0], part[1]));
        sum = both.x + both.y;
      }
      if (done >= 0) {
        // ---- the item before: its last product has had the time of this one's first weights
        if (done_any) {
          if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(o_bar + t), o_phase, abort_flag));
          if (!alive) break;
          o_phase ^= 1u;
          ptx::tc_fence_after_sync();
        }
        const int odd = output(items[done], done_any, done_sees, done_top, done_sum);
        if (__any_sync(~0u, odd)) row_by_row<T, D>(p, items[done], t, row, odd);
        __syncwarp();      // all lanes have read the item: its place is free
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(read_bar + done));
      }
      if (end) break;
      if (any) {
        announce(0);
        announce(1);
      }
      for (int s = skip + 1; s < steps; ++s) {
        if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(s_bar + t), s_phase, abort_flag));
        if (!alive) break;
        s_phase ^= 1u;
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) load(c);
        ptx::tmem_ld_wait();
        const int begin = (hi - 1 - s) * kRows;
        const bool masked = begin + kRows > first_limit;
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask(c, begin);
        }
        // Raises the maximum to `to`.  (The scores were issued behind the last product into O, so that is done.)
        const auto raise = [&](float to) {
          const float f = to == top ? 1.f : exp2_approx(top - to);
          top = to;
          sum *= f;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            ptx::tmem_ld_32x32b_x16(col_o + 16 * c, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st_32x32b_x16(col_o + 16 * c, o);
          }
        };
        part[0] = part[1] = pair(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = -INFINITY;
        weights(0, 48);
        // Where the sum of these weights, or the largest of the other scores, is out of reach they are done again.  (Maxima of
        // all scores instead, found beside the exponentials: 8192 tokens 463 us for 442.)
        const auto over = [&] {
          const float2 both = unpair(add2(part[0], part[1]));
          const float last = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2;
          return both.x + both.y > kMost || last > top + kMostLog2 || top == -INFINITY;
        };
        if (__any_sync(~0u, over() && limit > begin)) {
#pragma unroll
          for (int c = 0; c < kChecked / 16; ++c) load(c);
          ptx::tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int c = 0; c < kChecked / 16; ++c) mask(c, begin);
          }
#pragma unroll
          for (int i = 0; i < 2 * kChecked; i += 2) most[i & 2] = max3(most[i & 2], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          const float to = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.scale_log2;
          raise(marked(limit > begin ? fmaxf(to, top) : top));
          part[0] = part[1] = pair(0.f, 0.f);
          weights(0, kChecked);
        }
        ptx::tmem_st_32x32b_x32(col_s, *reinterpret_cast<uint32_t(*)[32]>(e16));
        ptx::tmem_st_32x32b_x16(col_s + 32, *reinterpret_cast<uint32_t(*)[16]>(e16 + 32));
        announce(0);
        weights(48, 64);
        ptx::tmem_st_32x32b_x16(col_s + 48, *reinterpret_cast<uint32_t(*)[16]>(e16 + 48));
        announce(1);
        const float2 both = unpair(add2(part[0], part[1]));
        sum += both.x + both.y;
      }
      done = slot, done_any = any, done_sees = limit > 0, done_top = top, done_sum = sum;
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

// The pieces of an item that was cut, in their order: a warp takes a row, a lane four dimensions (and the statistics of every 32nd
// piece).
constexpr int kJoinThreads = 256, kJoinBlocks = 8;      // blocks an SM: one wave, which ends at once where nothing was cut
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) attn_prefill_join_kernel(const PrefillParams p) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31, d = lane * 4, rows = p.header->joins * p.kv_heads * 2 * kRows;
  for (int all = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); all < rows; all += gridDim.x * (kJoinThreads / 32)) {
    const int r = all % (2 * kRows), row = r % kRows, kv = all / (2 * kRows) % p.kv_heads;
    const Item& it = p.joins[all / (2 * kRows) / p.kv_heads];
    const int query = it.first + r / kRows * p.tile_tokens + row / p.group;
    if (row >= p.tile_tokens * p.group || query >= it.n) continue;
    const auto at = [&](int c) { return (static_cast<int64_t>(it.slot + c) * p.kv_heads + kv) * 2 * kRows + r; };
    float top = -INFINITY;
    for (int c = lane; c < it.pieces; c += 32) top = fmaxf(top, p.part_ml[at(c)].x);
    for (int x = 16; x > 0; x /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
    const float base = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < it.pieces; c0 += 32) {
      const float2 ml = c0 + lane < it.pieces ? p.part_ml[at(c0 + lane)] : make_float2(-INFINITY, 0.f);
      const float weight = exp2_approx(ml.x - base);
      const int count = min(it.pieces - c0, 32);
      for (int c1 = 0; c1 < count; c1 += 8) {
        float4 v[8];      // all on their way at once
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = c1 + i < count && d < p.dim ? *reinterpret_cast<const float4*>(p.part_o + at(c0 + c1 + i) * D + d)
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = min(c1 + i, 31);
          const float f = __shfl_sync(~0u, weight, c), m = __shfl_sync(~0u, ml.x, c), s = __shfl_sync(~0u, ml.y, c);
          // A piece of which the row sees nothing: its sums may be anything.  (NaN scores beside hidden ones leave a maximum of -inf as well,
          // and a sum of NaN, which is the row's.)
          if (c1 + i >= count || (m == -INFINITY && s == 0.f)) continue;
          l += f * s;
          acc.x += v[i].x * f, acc.y += v[i].y * f, acc.z += v[i].z * f, acc.w += v[i].w * f;
        }
      }
    }
    const float inv = inverse(l);
    const int head = kv * p.group + row % p.group;
    if (d < p.dim)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (static_cast<int64_t>(it.row0 + query) * p.heads + head) * p.dim + d) =
          make_uint2(pack16<T>(acc.x * inv, acc.y * inv), pack16<T>(acc.z * inv, acc.w * inv));
  }
}

// What depends on the shapes and the hints alone.
struct Plan {
  int per_item, planned, split;
  int64_t items, units;      // at most
  size_t joins, ml, o;       // bytes of the workspace in front of each
  size_t bytes;
};

Plan make_plan(const b200q_attention& a) {
  Plan plan{};
  const int sms = sm_count(), d = a.dim <= 64 ? 64 : 128;
  plan.per_item = 2 * (kRows / (a.heads / a.kv_heads));
  // at most one item of each sequence is not full
  plan.items = std::min<int64_t>(a.tokens, a.tokens / plan.per_item + static_cast<int64_t>(a.sequences));
  // No item is cut where the longest has no more than an SM's share of all keys, each item having one tile of keys at
  // least; nor where it is short (64 queries over 2000 keys: whole 31 us, cut and joined 30; over 1100: 20 and 29).
  const int64_t longest = (static_cast<int64_t>(a.max_k) + kRows - 1) / kRows;
  plan.split = longest > 2 * kMinChunk && a.tokens / plan.per_item * a.kv_heads < sms * longest;
  plan.planned = plan.split || plan.items * a.kv_heads > sms;
  plan.units = plan.items + (plan.split ? 2 * sms : 0);
  if (!plan.planned) return plan;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  plan.joins = 256 + up(plan.units * sizeof(Item));
  plan.ml = plan.joins + (plan.split ? up(sms * sizeof(Item)) : 0);
  // an item that is cut has more than an SM's share, and at most twice as many pieces as shares: 2 pieces an SM
  plan.o = plan.ml + (plan.split ? up(2 * sms * 2 * kRows * sizeof(float2)) : 0);
  plan.bytes = plan.o + (plan.split ? static_cast<size_t>(2 * sms) * 2 * kRows * d * sizeof(float) : 0);
  return plan;
}

template <typename T, int D>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, PrefillParams p, const Plan& plan,
           cudaStream_t stream) {
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
  int launches = 1;
  p.ctas = static_cast<int>(plan.planned ? std::min<int64_t>(p.sms, plan.units * p.kv_heads) : plan.items * p.kv_heads);
  if (e == cudaSuccess && plan.planned) {
    e = launch_overlapped(MAX_SHARED, attn_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
    ++launches;
  }
  if (e == cudaSuccess)
    e = launch_overlapped(MAX_SHARED, kern, dim3(p.ctas), dim3(kThreads), smem, stream, tq, tk, tv, p);
  if (e == cudaSuccess && plan.split) {
    e = launch_overlapped(MAX_SHARED, attn_prefill_join_kernel<T, D>, dim3(p.sms * kJoinBlocks), dim3(kJoinThreads), 0, stream, p);
    ++launches;
  }
  if (e != cudaSuccess) {
    note_cuda_error(e);
    return B200Q_ERR_LAUNCH;
  }
  count_launch(launches);
  return B200Q_OK;
}

}  // namespace

size_t attn_prefill_workspace(const b200q_attention& a) { return make_plan(a).bytes; }

int launch_attn_prefill(const b200q_attention& a, void* workspace, int* status, cudaStream_t stream) {
  const Plan plan = make_plan(a);
  if (plan.units * a.kv_heads > INT_MAX / 2) return B200Q_ERR_BAD_SHAPE;
  PrefillParams p{};
  p.q = a.q, p.k = a.k, p.v = a.v;
  p.out = a.out;
  p.cu_q = a.cu_q, p.cu_k = a.cu_k, p.tables = a.tables, p.table_stride = a.table_stride;
  p.tokens = a.tokens, p.key_tokens = a.key_tokens, p.sequences = a.sequences;
  p.heads = a.heads, p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.dim = a.dim;
  p.pages = a.pages, p.page_size = a.page_size, p.table_width = a.table_width;
  p.tile_tokens = kRows / p.group;
  p.group_inverse = 65536 / p.group + 1;
  p.box_rows = kRows;
  while (a.page_size % p.box_rows != 0) p.box_rows /= 2;
  p.causal = a.causal;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = status;
  p.split = plan.split, p.sms = sm_count(), p.most_units = static_cast<int>(plan.units);
  if (plan.planned) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.header = reinterpret_cast<Header*>(ws);
    p.units = reinterpret_cast<Item*>(ws + 256);
    p.joins = reinterpret_cast<Item*>(ws + plan.joins);
    p.part_ml = reinterpret_cast<float2*>(ws + plan.ml);
    p.part_o = reinterpret_cast<float*>(ws + plan.o);
  }
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
    return bf ? launch<__nv_bfloat16, 64>(tq, tk, tv, p, plan, stream) : launch<__half, 64>(tq, tk, tv, p, plan, stream);
  return bf ? launch<__nv_bfloat16, 128>(tq, tk, tv, p, plan, stream) : launch<__half, 128>(tq, tk, tv, p, plan, stream);
}

}  // namespace b200q
