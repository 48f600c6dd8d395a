// Attention of one new token per sequence over a paged cache.
//
// o[b,h] = sum_j 2^(t_j - top) v_j / sum_j 2^(t_j - top),  t_j = scale log2(e) q[b,h] . k_j.
//
// Bound by memory: a key and a value of 2 D bytes each cost 4 D flops per query head that shares them.  So each is
// brought from memory once for all heads of its group, by TMA, and the products are mma.sync with the group as the
// short side (tcgen05 tiles have 128 rows: at 4 to 8 heads per key head they would compute on padding):
//   S^T [16 keys x 8 heads]  = K [16 x D] Q^T            K by ldmatrix, Q^T in registers
//   O^T [D x 8 heads]       += V^T [D x 16 keys] P^T      V by ldmatrix.trans; P^T is S^T turned by movmatrix
// A CTA has four such warps, each with 16 keys of every tile of 64 and running maximum, sum and O^T of its own (merged
// through shared memory at the end of a piece), and a warp that brings tiles through a ring.
//
// Work is divided by tiles, not by sequences: all tiles of all (sequence, key head) segments stand in one row, and each CTA
// takes the same number of neighbours, whatever the lengths are.  They are known on the device only, so each CTA adds them up
// itself.  Segments that a border cuts leave fp32 partial results (at most two pieces a CTA, so the workspace
// depends on the grid alone), which a second kernel, already resident, joins in a fixed order: no atomics, the same bits
// in every run.
//
// 64 sequences of 2000 to 8300 keys, 32 query and 8 key heads of 128: 204 us, 6.6 TB/s; one of 131071 keys: 90 us, 6.0 TB/s.
//
// The running maximum follows the scores lazily: it is raised (and sums rescaled) only when a score exceeds it by more than
// 8, so weights reach 2^8 at most; they are rounded to T with the same relative error wherever they stand.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "attn.h"
#include "attn_device.cuh"
#include "common.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

constexpr int kTile = 64;                       // keys
constexpr int kConsumers = 4;                   // warps, 16 keys of a tile each
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kRingBytes = 96 * 1024;           // two CTAs an SM
constexpr int kCtrlBytes = 256;
constexpr int kSegment = 1;                     // what a segment costs beside its tiles (queries, merging, output), in tiles
constexpr int kMinChunk = 6;                    // the least of a CTA, in tiles
constexpr int kUncut = 8;                       // tiles up to which a segment is not worth a join
constexpr float kLazy = 8.f;

struct DecodeParams {
  const void* q;
  int64_t q_token, q_head;
  void* out;
  const int32_t *lengths, *tables;
  int64_t table_stride;
  int sequences, heads, group, dim, pages, page_size, table_width;
  int segments;      // of a sequence: key heads x blocks of the heads that share one
  int head_blocks;
  int box_rows;
  int split;         // 0: no segment is cut
  float scale_log2;
  float* part_o;     // [2 CTAs][NT * 8][dim]
  float2* part_ml;   // [2 CTAs][NT * 8]: maximum, sum
  int4* joins;       // [CTAs]: sequence, segment, last CTA of a segment whose first piece is this CTA's; -1: none
  int* status;
};

__device__ __forceinline__ int clipped(int n, const DecodeParams& p) {
  return static_cast<int>(min(static_cast<int64_t>(min(max(n, 0), INT_MAX - kTile)),
                              static_cast<int64_t>(p.table_width) * p.page_size));
}
__device__ __forceinline__ int tiles_of(int length) { return max(1, (length + kTile - 1) / kTile); }

// The pieces of a CTA, one after another.  Every thread walks by itself.  A segment takes kSegment places in the row of all
// work, then one for each tile; a piece that is cut off before its first tile is none.
struct Walk {
  int b, seg, from, to, length;   // tiles [from, to) of the segment
  int ahead;                      // length of the next sequence
  int64_t left;                   // places behind this piece
  __device__ __forceinline__ bool whole() const { return from == 0 && to == tiles_of(length); }
  __device__ __forceinline__ void look_ahead(const DecodeParams& p) { ahead = b + 1 < p.sequences ? p.lengths[b + 1] : 0; }
  __device__ __forceinline__ bool cut(int at) {      // from this place of the segment on
    const int end = static_cast<int>(min(static_cast<int64_t>(tiles_of(length) + kSegment), at + left));
    left -= end - at;
    from = max(at - kSegment, 0);
    to = max(end - kSegment, 0);
    return to > from;
  }
  // the next piece: neighbouring tiles, or, where no segment is cut, every gridDim.x-th segment; false: none
  __device__ __forceinline__ bool next(const DecodeParams& p) {
    if (p.split) {
      if (left <= 0) return false;
      if (++seg == p.segments) {
        seg = 0;
        ++b;
        length = clipped(ahead, p);
        look_ahead(p);
      }
    } else {
      const int64_t at = static_cast<int64_t>(b) * p.segments + seg + gridDim.x;
      b = static_cast<int>(min(at / p.segments, static_cast<int64_t>(p.sequences)));
      if (b == p.sequences) return false;
      seg = static_cast<int>(at % p.segments);
      length = clipped(p.lengths[b], p);
      left = INT_MAX;
    }
    return cut(0);
  }
};

// The warps' results of a piece, eight heads at a time: a row of D sums, then maximum and sum of the weights.
template <int D>
constexpr int comb_bytes() { return kConsumers * 8 * (D + 4) * 4; }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2)
attn_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const DecodeParams p) {
  constexpr int kHalves = D / 64;
  constexpr int kSide = kTile * D * 2;                 // bytes of a tile's keys
  constexpr int kStages = kRingBytes / (2 * kSide);
  extern __shared__ __align__(1024) uint8_t smem[];
  float* comb = reinterpret_cast<float*>(smem + kRingBytes);                       // [warp][8 heads][D + 4]
  uint8_t* ctrl = smem + kRingBytes + comb_bytes<D>();
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty_bar = full_bar + kStages;
  Walk& s_walk = *reinterpret_cast<Walk*>(empty_bar + kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(&s_walk + 1);
  int64_t* scan = reinterpret_cast<int64_t*>(comb);                                // before the ring starts
  static_assert(16 * kStages + sizeof(Walk) + sizeof(int) <= kCtrlBytes && sizeof(Walk) % 8 == 0, "control words");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_base = ptx::smem_u32(smem);
  if ((smem_base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 0x200);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(full_bar + s), 1);
      ptx::mbar_init(ptx::smem_u32(empty_bar + s), kConsumers);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::tma_prefetch_desc(&tmap_k);
    ptx::tma_prefetch_desc(&tmap_v);
  }
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();

  // Tiles in front of each thread's share of the sequences.
  const int per = (p.sequences + kThreads - 1) / kThreads, b0 = threadIdx.x * per;
  int64_t mine = 0;
  for (int b = b0; b < min(b0 + per, p.sequences); ++b) mine += tiles_of(clipped(p.lengths[b], p)) + kSegment;
  int64_t upto = mine;
  for (int x = 1; x < 32; x *= 2) {
    const int64_t o = __shfl_up_sync(~0u, upto, x);
    if (lane >= x) upto += o;
  }
  if (lane == 31) scan[warp] = upto;
  if (threadIdx.x == 0) s_walk.left = -1;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w <= kConsumers; ++w) {
    if (w == warp) upto += total;
    total += scan[w];
  }
  total *= p.segments;
  int64_t first = (upto - mine) * p.segments;
  int64_t chunk, start;
  if (p.split) {
    chunk = max((total + gridDim.x - 1) / static_cast<int64_t>(gridDim.x), static_cast<int64_t>(kMinChunk));
    start = blockIdx.x * chunk;
    if (start >= first && start < first + mine * p.segments) {     // one thread
      int b = b0, places;
      while (true) {
        s_walk.length = clipped(p.lengths[b], p);
        places = tiles_of(s_walk.length) + kSegment;
        if (start < first + static_cast<int64_t>(places) * p.segments) break;
        first += static_cast<int64_t>(places) * p.segments;
        ++b;
      }
      s_walk.b = b;
      s_walk.seg = static_cast<int>((start - first) / places);
      s_walk.from = static_cast<int>((start - first) % places);
      s_walk.left = min(chunk, total - start);
      s_walk.look_ahead(p);
    }
  } else if (threadIdx.x == 0) {
    // whole segments, blockIdx.x, blockIdx.x + gridDim.x, ...: `left` counts for one at a time
    s_walk.b = blockIdx.x / p.segments;
    s_walk.seg = blockIdx.x % p.segments;
    s_walk.from = 0;
    s_walk.left = s_walk.b < p.sequences ? INT_MAX : -1;
    if (s_walk.b < p.sequences) s_walk.length = clipped(p.lengths[s_walk.b], p);
  }
  __syncthreads();
  Walk w = s_walk;
  if (p.split && threadIdx.x == 0) {
    // the CTA's last segment, if it goes on behind the CTA's last tile, and begins here
    p.joins[blockIdx.x].x = -1;
  }
  const bool any = w.left > 0;
  __syncthreads();   // comb (the scan) is free
  if (any) {
    w.cut(w.from);      // (never empty: a CTA's places are more than kSegment or reach the row's end)
    int stage = 0;
    uint32_t phase = 0;
    bool go = true;
    if (warp == kConsumers) {
      // ------------------------------------------------------------------ producer
      bool alive = true;
      const int boxes = kTile / p.box_rows;            // of a tile; a lane holds the page of one box
      int page = 0, first_pages = -1;                  // of which sequence they are the first ones
      while (go) {
        const int kv = w.seg / p.head_blocks;
        const int32_t* table = p.tables + w.b * p.table_stride;
        int batch = -1;
        // a sequence's key heads have the same first pages
        if (w.from == 0 && w.b == first_pages) batch = 0;
        const int last = w.length == 0 ? w.from : w.to;
        for (int u = w.from; u < last; ++u) {
          // pages of the next 32 boxes at a time
          if ((u - w.from) * boxes / 32 != batch) {
            batch = (u - w.from) * boxes / 32;
            first_pages = u == 0 ? w.b : -1;
            const int64_t pos = static_cast<int64_t>(u) * kTile + lane * p.box_rows;
            if (pos < w.length) {
              page = table[pos / p.page_size];
              if (page < 0 || page >= p.pages) {
                atomicCAS(p.status, 0, 0xa01);
                page = p.pages;                       // outside: the copy brings zeros
              }
            }
          }
          if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(empty_bar + stage), phase ^ 1u, abort_flag));
          const int begin = u * kTile, held = min(boxes, (w.length - begin + p.box_rows - 1) / p.box_rows);
          const int mine_page = __shfl_sync(~0u, page, ((u - w.from) * boxes + lane) & 31);
          const uint32_t bar = ptx::smem_u32(full_bar + stage);
          if (lane == 0 && alive) ptx::mbar_arrive_expect_tx(bar, held * p.box_rows * D * 4);
          __syncwarp();
          if (lane < held && alive) {
            const int at = (begin + lane * p.box_rows) % p.page_size;
            const uint32_t dst = smem_base + stage * 2 * kSide + lane * p.box_rows * 128;
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              ptx::tma_load_4d(dst + h * kTile * 128, &tmap_k, bar, h * 64, kv, at, mine_page);
              ptx::tma_load_4d(dst + kSide + h * kTile * 128, &tmap_v, bar, h * 64, kv, at, mine_page);
            }
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        go = w.next(p);
      }
      __syncwarp();
      if (lane == 0) {
        if (*abort_flag != 0) ptx::drain_ring(full_bar, kStages, stage, phase);
      }
    } else {
      // ------------------------------------------------------------------ consumers
      const int gid = lane >> 2, tid = lane & 3;
      bool alive = true;
      // Q^T as the B operand: lane holds dimensions 16 k + 2 tid, + 1, + 8, + 9 of head gid
      uint32_t qf[NT][D / 16][2];
      const auto load_queries = [&](const Walk& w) {
        const int block = w.seg % p.head_blocks, head0 = w.seg / p.head_blocks * p.group + block * 8 * NT;
        const int rows = p.group - block * 8 * NT;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const T* q = static_cast<const T*>(p.q) + w.b * p.q_token + (head0 + 8 * t + gid) * p.q_head;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int d = 16 * k + 8 * i + 2 * tid;
              qf[t][k][i] = 8 * t + gid < rows && d < p.dim ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
            }
        }
      };
      load_queries(w);
      while (go) {
        const int kv = w.seg / p.head_blocks, head0 = kv * p.group + (w.seg % p.head_blocks) * 8 * NT;
        const int rows = min(8 * NT, p.group - (w.seg % p.head_blocks) * 8 * NT);
        float o[NT][D / 16][4], top[NT][2], sum[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          top[t][0] = top[t][1] = -INFINITY;
          sum[t][0] = sum[t][1] = 0.f;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) o[t][k][0] = o[t][k][1] = o[t][k][2] = o[t][k][3] = 0.f;
        }
        const int last = w.length == 0 ? w.from : w.to;
        for (int u = w.from; u < last; ++u) {
          if (alive) alive = ptx::warp_all(ptx::mbar_wait(ptx::smem_u32(full_bar + stage), phase, abort_flag));
          const uint32_t keys = smem_base + stage * 2 * kSide, values = keys + kSide;
          // rows of matrices 0, 1: keys 0-7, 8-15 (K) or dimensions 0-7, 8-15 (V); 2, 3: the other eight of the other
          const int krow = warp * 16 + (lane & 15);
          const int vrow = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
          const int behind = w.length - u * kTile - warp * 16;      // this warp's keys from here on do not exist
          if (alive) {
            if (behind < 16) {
              // what a page holds behind the sequence's end may be anything, and 0 * NaN is NaN
              for (int r = max(behind, 0); r < 16; ++r)
                for (int c = lane; c < D / 8; c += 32)
                  *reinterpret_cast<uint4*>(smem + (values - smem_base) + (c >> 3) * kTile * 128 + (warp * 16 + r) * 128 +
                                            (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
              __syncwarp();
            }
            float s[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t a[4];
              const int piece = (2 * k + (lane >> 4)) & 7;
              ldmatrix_x4(a, keys + (k >> 2) * kTile * 128 + krow * 128 + ((piece ^ (krow & 7)) << 4));
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_16<T>(s[t], a[0], a[1], a[2], a[3], qf[t][k][0], qf[t][k][1]);
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
              for (int i = 0; i < 4; ++i)      // (key gid, head 2 tid), (gid, 2 tid + 1), (gid + 8, ...)
                s[t][i] = gid + 8 * (i >> 1) < behind ? s[t][i] * p.scale_log2 : -INFINITY;
              const float t0 = fmaxf(s[t][0], s[t][2]), t1 = fmaxf(s[t][1], s[t][3]);
              if (__any_sync(~0u, t0 > top[t][0] + kLazy || t1 > top[t][1] + kLazy)) {
                float n0 = t0, n1 = t1;
#pragma unroll
                for (int x = 4; x < 32; x *= 2) {
                  n0 = fmaxf(n0, __shfl_xor_sync(~0u, n0, x));
                  n1 = fmaxf(n1, __shfl_xor_sync(~0u, n1, x));
                }
                n0 = fmaxf(n0, top[t][0]);
                n1 = fmaxf(n1, top[t][1]);
                const float f0 = n0 == top[t][0] ? 1.f : exp2_approx(top[t][0] - n0);
                const float f1 = n1 == top[t][1] ? 1.f : exp2_approx(top[t][1] - n1);
                top[t][0] = n0;
                top[t][1] = n1;
                sum[t][0] *= f0;
                sum[t][1] *= f1;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  o[t][k][0] *= f0;
                  o[t][k][1] *= f1;
                  o[t][k][2] *= f0;
                  o[t][k][3] *= f1;
                }
              }
              const float m0 = top[t][0] == -INFINITY ? 0.f : top[t][0], m1 = top[t][1] == -INFINITY ? 0.f : top[t][1];
              const float p0 = exp2_approx(s[t][0] - m0), p1 = exp2_approx(s[t][1] - m1);
              const float p2 = exp2_approx(s[t][2] - m0), p3 = exp2_approx(s[t][3] - m1);
              sum[t][0] += p0 + p2;
              sum[t][1] += p1 + p3;
              pf[t][0] = movmatrix_trans(pack16<T>(p0, p1));
              pf[t][1] = movmatrix_trans(pack16<T>(p2, p3));
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t a[4];
              const int piece = (2 * k + ((lane >> 3) & 1)) & 7;
              ldmatrix_x4_trans(a, values + (k >> 2) * kTile * 128 + vrow * 128 + ((piece ^ (vrow & 7)) << 4));
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_16<T>(o[t][k], a[0], a[1], a[2], a[3], pf[t][0], pf[t][1]);
            }
            if (behind < 16) ptx::fence_proxy_async_smem();      // the zeros, before the next copy into this place
          }
          __syncwarp();
          if (lane == 0 && alive) ptx::mbar_arrive(ptx::smem_u32(empty_bar + stage));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }

        // ---- the next piece's queries, on their way while this one's results are merged
        Walk next = w;
        go = next.next(p);
        if (go) load_queries(next);
        // ---- the four warps' results of this piece
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int x = 4; x < 32; x *= 2) sum[t][i] += __shfl_xor_sync(~0u, sum[t][i], x);
        const bool whole = w.whole();
        const int part = blockIdx.x * 2 + (w.from == 0 ? 1 : 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              comb[(warp * 8 + 2 * tid + (i & 1)) * (D + 4) + 16 * k + gid + 8 * (i >> 1)] = o[t][k][i];
          if (gid < 2)
            *reinterpret_cast<float2*>(comb + (warp * 8 + 2 * tid + gid) * (D + 4) + D) =
                make_float2(gid == 0 ? top[t][0] : top[t][1], gid == 0 ? sum[t][0] : sum[t][1]);
          ptx::named_bar_sync(1, kConsumers * 32);
          // a thread: 4 dimensions of one head at a time
          for (int e = threadIdx.x; e < 8 * (D / 4); e += kConsumers * 32) {
            const int h = e / (D / 4), d = e % (D / 4) * 4, row = 8 * t + h;
            if (row >= rows || d >= p.dim) continue;
            float m = -INFINITY, l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) m = fmaxf(m, comb[(x * 8 + h) * (D + 4) + D]);
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) {
              const float2 ml = *reinterpret_cast<const float2*>(comb + (x * 8 + h) * (D + 4) + D);
              const float f = exp2_approx(ml.x - base);
              const float4 v = *reinterpret_cast<const float4*>(comb + (x * 8 + h) * (D + 4) + d);
              l += f * ml.y;
              acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            }
            if (whole) {
              const float inv = inverse(l);
              uint2 packed = make_uint2(pack16<T>(acc.x * inv, acc.y * inv), pack16<T>(acc.z * inv, acc.w * inv));
              *reinterpret_cast<uint2*>(static_cast<T*>(p.out) +
                                        (static_cast<int64_t>(w.b) * p.heads + head0 + row) * p.dim + d) = packed;
            } else {
              *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(part) * 8 * NT + row) * D + d) = acc;
              if (d == 0) p.part_ml[part * 8 * NT + row] = make_float2(m, l);
            }
          }
          ptx::named_bar_sync(1, kConsumers * 32);
        }
        if (!whole && w.from == 0 && threadIdx.x == 0) {
          const int64_t behind = tiles_of(w.length) - w.to;      // tiles of the segment in the CTAs behind this one
          p.joins[blockIdx.x] = make_int4(w.b, w.seg, static_cast<int>(blockIdx.x + (behind + chunk - 1) / chunk), 0);
        }
        w = next;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicCAS(p.status, 0, 0x900 | (static_cast<int>(blockIdx.x) << 12));
}

// One block per CTA of the first kernel and head: the pieces of the segment that begins with that CTA's last one, a warp each,
// four dimensions a lane; then the warps' sums in order.
constexpr int kJoinWarps = 4;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const DecodeParams p) {
  __shared__ float4 acc_s[kJoinWarps][32];
  __shared__ float2 ml_s[kJoinWarps];
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int4 join = p.joins[blockIdx.x];
  if (join.x < 0) return;
  const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block = join.y % p.head_blocks, kv = join.y / p.head_blocks;
  if (block * 8 * NT + row >= p.group) return;
  const int first = blockIdx.x, last = join.z, d = lane * 4;
  const bool mine = d < p.dim;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = first + warp; c <= last; c += kJoinWarps) {
    const int64_t part = static_cast<int64_t>(c) * 2 + (c == first ? 1 : 0);
    const float2 ml = p.part_ml[part * 8 * NT + row];
    const float4 v = mine ? *reinterpret_cast<const float4*>(p.part_o + (part * 8 * NT + row) * D + d) : acc;
    const float n = fmaxf(m, ml.x), base = n == -INFINITY ? 0.f : n;
    const float f = exp2_approx(m - base), g = exp2_approx(ml.x - base);
    m = n;
    l = l * f + ml.y * g;
    acc.x = acc.x * f + v.x * g, acc.y = acc.y * f + v.y * g;
    acc.z = acc.z * f + v.z * g, acc.w = acc.w * f + v.w * g;
  }
  acc_s[warp][lane] = acc;
  if (lane == 0) ml_s[warp] = make_float2(m, l);
  __syncthreads();
  if (warp != 0 || !mine) return;
#pragma unroll
  for (int x = 0; x < kJoinWarps; ++x) m = fmaxf(m, ml_s[x].x);
  const float base = m == -INFINITY ? 0.f : m;
  l = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int x = 0; x < kJoinWarps; ++x) {
    const float f = exp2_approx(ml_s[x].x - base);
    const float4 v = acc_s[x][lane];
    l += ml_s[x].y * f;
    acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
  }
  const float inv = inverse(l);
  const int head = kv * p.group + block * 8 * NT + row;
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (static_cast<int64_t>(join.x) * p.heads + head) * p.dim + d) =
      make_uint2(pack16<T>(acc.x * inv, acc.y * inv), pack16<T>(acc.z * inv, acc.w * inv));
}

// What depends on the shapes alone.
struct Plan {
  int d, nt, head_blocks, grid, split;
  size_t joins, ml, o;      // bytes
};

Plan make_plan(const b200q_attention& a) {
  Plan plan{};
  const int group = a.heads / a.kv_heads;
  plan.d = a.dim <= 64 ? 64 : 128;
  plan.nt = group <= 8 ? 1 : 2;
  plan.head_blocks = (group + 8 * plan.nt - 1) / (8 * plan.nt);
  const int64_t segments = static_cast<int64_t>(a.sequences) * a.kv_heads * plan.head_blocks;
  const int64_t most = (static_cast<int64_t>(a.table_width) * a.page_size + kTile - 1) / kTile;   // tiles of a segment
  const int64_t ctas = sm_count() * 2;
  plan.split = most > kUncut;
  plan.grid = static_cast<int>(std::min(ctas, plan.split ? segments * ((most + kSegment + kMinChunk - 1) / kMinChunk) : segments));
  if (plan.split) {
    plan.joins = (plan.grid * sizeof(int4) + 255) / 256 * 256;
    plan.ml = (static_cast<size_t>(plan.grid) * 2 * 8 * plan.nt * sizeof(float2) + 255) / 256 * 256;
    plan.o = static_cast<size_t>(plan.grid) * 2 * 8 * plan.nt * plan.d * sizeof(float);
  }
  return plan;
}

template <typename T, int D, int NT>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p, const Plan& plan, cudaStream_t stream) {
  constexpr int smem = kRingBytes + comb_bytes<D>() + kCtrlBytes;
  static_assert(2 * (smem + kCtaSharedExtra) <= kSmSharedBytes, "two CTAs an SM");
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  auto kern = attn_decode_kernel<T, D, NT>;
  cudaError_t e = cudaSuccess;
  if (dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) attr_set[dev] = true;
  }
  if (e == cudaSuccess)
    e = launch_overlapped(MAX_SHARED, kern, dim3(plan.grid), dim3(kThreads), smem, stream, tk, tv, p);
  if (e == cudaSuccess) {
    count_launch();
    if (plan.split) {
      e = launch_overlapped(MAX_SHARED, attn_join_kernel<T, D, NT>, dim3(plan.grid, std::min(8 * NT, p.group)),
                            dim3(kJoinWarps * 32), 0, stream, p);
      if (e == cudaSuccess) count_launch();
    }
  }
  if (e != cudaSuccess) {
    note_cuda_error(e);
    return B200Q_ERR_LAUNCH;
  }
  return B200Q_OK;
}

template <typename T>
int launch_sized(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p, const Plan& plan, cudaStream_t stream) {
  if (plan.d == 64)
    return plan.nt == 1 ? launch<T, 64, 1>(tk, tv, p, plan, stream) : launch<T, 64, 2>(tk, tv, p, plan, stream);
  return plan.nt == 1 ? launch<T, 128, 1>(tk, tv, p, plan, stream) : launch<T, 128, 2>(tk, tv, p, plan, stream);
}

}  // namespace

bool make_key_map(const b200q_view& x, const b200q_attention& a, uint32_t box_rows, CUtensorMap* out) {
  const bool paged = a.page_size > 0;
  const uint64_t size[4] = {static_cast<uint64_t>(a.dim), static_cast<uint64_t>(a.kv_heads),
                            static_cast<uint64_t>(paged ? a.page_size : std::max(a.key_tokens, 1)),
                            static_cast<uint64_t>(paged ? a.pages : 1)};
  int64_t stride[3] = {x.head, x.token, x.page};
  for (int i = 0; i < 3; ++i)
    if (size[i + 1] == 1) stride[i] = (a.dim + 7) / 8 * 8;      // says nothing, but has to be valid
  const uint32_t box[4] = {64, 1, box_rows, 1};
  return make_tensor_map_16(x.data, 4, size, stride, box, out);
}

size_t attn_decode_workspace(const b200q_attention& a) {
  const Plan plan = make_plan(a);
  return plan.joins + plan.ml + plan.o;
}

int launch_attn_decode(const b200q_attention& a, void* workspace, int* status, cudaStream_t stream) {
  const Plan plan = make_plan(a);
  DecodeParams p{};
  p.q = a.q.data, p.q_token = a.q.token, p.q_head = a.q.head;
  p.out = a.out;
  p.lengths = a.lengths, p.tables = a.tables, p.table_stride = a.table_stride;
  p.sequences = a.sequences, p.heads = a.heads, p.group = a.heads / a.kv_heads, p.dim = a.dim;
  p.pages = a.pages, p.page_size = a.page_size, p.table_width = a.table_width;
  p.head_blocks = plan.head_blocks, p.segments = a.kv_heads * plan.head_blocks;
  p.box_rows = 16;
  while (p.box_rows < kTile && a.page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
  p.split = plan.split;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.joins = reinterpret_cast<int4*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + plan.joins);
  p.part_o = reinterpret_cast<float*>(ws + plan.joins + plan.ml);
  p.status = status;
  CUtensorMap tk, tv;
  if (!make_key_map(a.k, a, p.box_rows, &tk) || !make_key_map(a.v, a, p.box_rows, &tv)) return B200Q_ERR_LAUNCH;
  return a.dtype == B200Q_DTYPE_BF16 ? launch_sized<__nv_bfloat16>(tk, tv, p, plan, stream)
                                     : launch_sized<__half>(tk, tv, p, plan, stream);
}

}  // namespace b200q
