// Attention of single query tokens over a paged key-value cache.
//
// Query i (position pos of request row) sees keys j in [max(0, pos - window), pos]:
//   o = sum_j softmax_j(scale * q . k_j - slope_h * (pos - j)) v_j
// K and V are read once each: 4 * D bytes per key and KV head for 4 * D * G flops (the G query heads that
// share a KV head), at most 16 flops per byte for G = 16, so HBM bandwidth is the bound and the design is
// about keeping enough bytes in flight on every SM whatever the lengths are.
//
// * Work is cut into tiles of 64 keys of one KV head (item = query x KV head). The kernel computes, from the
//   positions on the device, how many tiles there are and gives every CTA an equal contiguous share, so one
//   request of any length, or a batch of mixed lengths, fills the GPU without a plan from the host (and a
//   CUDA graph follows the lengths). A CTA whose share starts or ends inside an item leaves an fp32 partial
//   (running max, sum, unnormalized output); a second, small kernel joins an item's partials in tile order,
//   so results do not depend on timing.
// * One producer warp reads the block table 32 entries at a time and issues one TMA box per page for K and
//   one for V (128-byte swizzle, so the fragment loads are free of bank conflicts) into a ring of stages. Pages
//   that hold no visible key are requested out of range: TMA fills zeros and reads nothing, and a corrupt
//   table entry cannot read outside the pool.
// * Four consumer warps split a tile: RW warps over query rows (16 each), 4 / RW over keys. Each keeps its own
//   running max, sum and output in registers, so there is no exchange until an item ends, when the warps'
//   results are merged through the item's last stage. Products run on mma.sync m16n8k16: with at most 16 (64)
//   live rows an M = 128 tcgen05 tile would be mostly padding, and the tensor pipe is not the bound.
// * P is split into two 16-bit terms (p = hi + lo) for the second product, so probabilities keep 16 bits of
//   precision instead of 8 (bf16) at no cost in time; scores, sums and outputs are fp32.
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "paged.cuh"

namespace mint {
namespace paged {

constexpr int kTile = 64;          // keys per tile
constexpr int kWarps = 4;          // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kMinTiles = 1;       // a share is at least this many tiles
constexpr int kJoinThreads = 1024;

template <int D, int RW>
struct Config {
  static constexpr int kRows = 16 * RW;  // query rows per item
  static constexpr int kKvBytes = kTile * D * 2;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kStageBytes = (2 * kKvBytes + kQBytes + 1023) / 1024 * 1024;
  // two CTAs per SM where three stages fit twice, else one
  static constexpr int kControl = 2048;  // barriers, tile descriptions, merge statistics, base alignment
  static constexpr int kHalf = 113 * 1024, kFull = 227 * 1024;
  static constexpr bool kTwo = (kHalf - kControl) / kStageBytes >= 3;
  static constexpr int kFit = ((kTwo ? kHalf : kFull) - kControl) / kStageBytes;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static_assert(kStages >= 2 && kSmem + 1024 <= kFull, "shared memory");
};

struct TileInfo {  // the tile in a stage, for the consumers
  int query, group;  // item: query and KV head * row groups + row group
  int key0, lo, hi, pos;
  int out;    // partial slot, or -1: write the output
  int flags;  // 1: first tile of a piece (the stage holds Q), 2: last
};

struct AttnParams {
  const void* q;  // [N, Hq, D]
  void* o;
  const int* tables;     // [B, W], row stride tstride
  const int* positions;  // [N]
  const int* rows;       // [N] or null (row i = i)
  const float* slopes;   // [Hq] or null
  float* part_o;         // [2 * grid][rows][D]
  float2* part_ml;       // [2 * grid][rows]
  int4* joins;           // [grid] (query, group, first partial's CTA, partials) or partials = 0
  uint32_t* status;
  long long tstride;
  int N, B, W, Hq, Hkv, G, groups, part_rows, n_pages, page_shift, window;
  float scale_log2;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (a, b) = hi + lo in two packed 16-bit pairs; lo holds what rounding to hi lost
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(a, b);
  const float2 f = bf16x2_to_float2(hi);
  lo = pack_bf16x2(a - f.x, b - f.y);
}
template <>
__device__ __forceinline__ void split2<__half>(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, uint64_t* bar, int line, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(line), "r"(0), "r"(head), "r"(page)
      : "memory");
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Keys [lo, hi) that query n sees (hi = 0: none) and its table row.
struct Span {
  int row, lo, hi, pos;
  __device__ __forceinline__ int first() const { return lo / kTile; }
  __device__ __forceinline__ int tiles() const { return hi > 0 ? (hi - 1) / kTile - lo / kTile + 1 : 0; }
};
__device__ __forceinline__ Span span_of(const AttnParams& p, int row, int pos) {
  Span s{row, 0, 0, pos};
  if (row < 0 || row >= p.B || pos < 0) return s;
  s.pos = min(pos, static_cast<int>((static_cast<long long>(p.W) << p.page_shift) - 1));
  s.hi = s.pos + 1;
  s.lo = p.window >= 0 ? max(0, s.pos - p.window) : 0;
  return s;
}
__device__ __forceinline__ Span span_at(const AttnParams& p, int n) {
  return span_of(p, p.rows != nullptr ? p.rows[n] : n, p.positions[n]);
}

template <typename T, int D, int RW>
__global__ void __launch_bounds__(kThreads, Config<D, RW>::kTwo ? 2 : 1)
    attend_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, AttnParams p) {
  using C = Config<D, RW>;
  extern __shared__ uint8_t s_raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages], merge;
  __shared__ TileInfo info[C::kStages];
  __shared__ float2 s_ml[kWarps][16];
  __shared__ long long s_sum[kWarps + 1], s_off, s_total;
  __shared__ int s_query, s_abort;
  uint8_t* stages = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x;
  const int per_query = p.Hkv * p.groups;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    mbar_init(&merge, kWarps);
    s_abort = 0;
    s_query = 0;
    s_off = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  // this CTA's share of the tiles: totals by a scan over the queries
  const int chunk = (p.N + kThreads - 1) / kThreads;
  const int n0 = min(p.N, tid * chunk), n1 = min(p.N, n0 + chunk);
  long long mine = 0;
  for (int n = n0; n < n1; ++n) mine += span_at(p, n).tiles();
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  long long before = inc - mine, total = 0;
#pragma unroll
  for (int w = 0; w <= kWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const long long all = total * per_query;
  const long long ctas = max(1ll, min(static_cast<long long>(gridDim.x), (all + kMinTiles - 1) / kMinTiles));
  const long long t0 = cta < ctas ? all * cta / ctas : all, t1 = cta < ctas ? all * (cta + 1) / ctas : all;
  if (t1 > t0) {
    const long long u = t0 / per_query;
    if (before <= u && u < before + mine) {
      long long at = before;
      for (int n = n0; n < n1; ++n) {
        const int c = span_at(p, n).tiles();
        if (u < at + c) {
          s_query = n;
          s_off = t0 - at * per_query;
          break;
        }
        at += c;
      }
    }
  }
  __syncthreads();
  const long long count = t1 - t0;

  if (warp == kWarps) {
    // ------------------------------------------------------------------------------- producer
    int n = s_query, stage = 0;
    long long off = s_off, left = count;
    uint32_t phase = 0;
    int4 join = make_int4(0, 0, 0, 0);
    const int rows_in_box = min(1 << p.page_shift, kTile);
    const int boxes = kTile / rows_in_box;
    bool ok = true, bad = false;
    long long issued = 0;
    while (left > 0 && ok) {
      const Span s = span_at(p, n);
      const int tiles = s.tiles();
      if (off >= static_cast<long long>(tiles) * per_query) {
        ++n;
        off = 0;
        continue;
      }
      bad |= p.positions[n] != s.pos;
      const int group = static_cast<int>(off / tiles), at = static_cast<int>(off - static_cast<long long>(group) * tiles);
      const int len = static_cast<int>(min(left, static_cast<long long>(tiles - at)));
      const int kv_head = group / p.groups, row0 = (group - kv_head * p.groups) * C::kRows;
      const int live_rows = min(C::kRows, p.G - row0);
      int out = -1;
      if (at > 0) {
        out = 2 * cta;
      } else if (len < tiles) {
        out = 2 * cta + 1;
        // the last tile's owner: the largest c with all * c / ctas <= tile
        const long long last = t1 - left + tiles - 1;
        join = make_int4(n, group, cta, static_cast<int>(((last + 1) * ctas - 1) / all) - cta + 1);
      }
      const int* table = p.tables + s.row * p.tstride;
      const int last_page = s.pos >> p.page_shift;
      int base = ((s.first() + at) * kTile) >> p.page_shift;
      int entry = base + lane <= last_page ? table[base + lane] : -1;
      for (int i = 0; i < len; ++i) {
        const int key0 = (s.first() + at + i) * kTile;
        const int page0 = key0 >> p.page_shift;
        if (page0 >= base + 32) {
          base = page0;
          entry = base + lane <= last_page ? table[base + lane] : -1;
        }
        int page = __shfl_sync(0xffffffffu, entry, (page0 - base + lane) & 31);
        const int number = page0 + lane;
        if (number > last_page || ((number + 1) << p.page_shift) <= s.lo) {
          page = p.n_pages;  // nothing visible in it: zero fill
        } else if (lane < boxes && (page < 0 || page >= p.n_pages)) {
          bad = true;
          page = p.n_pages;
        }
        if (!mbar_wait_warp(&empty[stage], phase ^ 1u, p.status, kStatusTimeoutAttention, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* buf = stages + stage * C::kStageBytes;
        if (lane == 0) {
          TileInfo& t = info[stage];
          t.query = n;
          t.group = group;
          t.key0 = key0;
          t.lo = s.lo;
          t.hi = s.hi;
          t.pos = s.pos;
          t.out = out;
          t.flags = (i == 0 ? 1 : 0) | (i == len - 1 ? 2 : 0);
          mbar_arrive_expect_tx(&full[stage], 2 * C::kKvBytes + (i == 0 ? live_rows * D * 2 : 0));
        }
        __syncwarp();
        if (lane < boxes) {
          const int line = boxes == 1 ? key0 & ((1 << p.page_shift) - 1) : 0;
          tma_load_page(buf + lane * rows_in_box * D * 2, &tk, &full[stage], line, kv_head, page);
          tma_load_page(buf + C::kKvBytes + lane * rows_in_box * D * 2, &tv, &full[stage], line, kv_head, page);
        }
        if (i == 0 && lane == 0) {
          const T* q = static_cast<const T*>(p.q) + (static_cast<long long>(n) * p.Hq + kv_head * p.G + row0) * D;
          bulk_load(buf + 2 * C::kKvBytes, q, live_rows * D * 2, &full[stage]);
        }
        ++issued;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      off += len;
      left -= len;
    }
    if (lane == 0) p.joins[cta] = join;
    if (__any_sync(0xffffffffu, bad) && lane == 0) record_status(p.status, kStatusBadArgument);
    if (!ok) {  // given up: no copy may land after the CTA is gone
      for (int i = 0; i < C::kStages && i < issued; ++i) {
        const int back = stage - 1 - i;
        const int st = back < 0 ? back + C::kStages : back;
        const uint32_t ph = back < 0 ? phase ^ 1u : phase;
        mbar_wait_warp(&full[st], ph, p.status, kStatusTimeoutAttention, nullptr);
      }
    }
    return;
  }

  // ----------------------------------------------------------------------------------- consumers
  for (int n = cta; n < p.N; n += gridDim.x) {  // queries without keys: zeros
    if (span_at(p, n).hi > 0) continue;
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + static_cast<long long>(n) * p.Hq * D);
    for (int i = tid; i < p.Hq * D / 8; i += 32 * kWarps) o[i] = make_uint4(0, 0, 0, 0);
  }
  const int rw = warp % RW, kw = warp / RW;
  const int box_shift = min(p.page_shift, 6), box_rows = 1 << box_shift;
  const uint32_t half_stride = box_rows * 128;  // bytes between 64-column parts of a box
  auto line_offset = [&](int r) { return static_cast<uint32_t>((r >> box_shift) * box_rows * D * 2 + (r & (box_rows - 1)) * 128); };
  uint32_t k_line[RW], v_line[RW];
#pragma unroll
  for (int b = 0; b < RW; ++b) {
    const int r0 = (kw * RW + b) * 16;
    k_line[b] = line_offset(r0 + (lane & 7) + ((lane >> 4) << 3));
    v_line[b] = line_offset(r0 + (lane & 15));
  }
  const uint32_t k_chunk = ((lane >> 3) & 1) ^ (lane & 7), v_chunk = (lane >> 4) ^ (lane & 7);
  const uint32_t base_addr = smem_u32(stages);

  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, slope[2] = {0.f, 0.f};
  int stage = 0;
  uint32_t phase = 0, merge_phase = 0;
  for (long long it = 0; it < count; ++it) {
    if (!mbar_wait_warp(&full[stage], phase, p.status, kStatusTimeoutAttention, abort_flag)) return;
    const TileInfo t = info[stage];
    const uint32_t k_addr = base_addr + stage * C::kStageBytes, v_addr = k_addr + C::kKvBytes;
    const int kv_head = t.group / p.groups, row0 = (t.group - kv_head * p.groups) * C::kRows;
    if (t.flags & 1) {
      const uint32_t q_addr = k_addr + 2 * C::kKvBytes + (rw * 16 + (lane & 15)) * (D * 2) + (lane >> 4) * 16;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) ldsm4(qf[ks], q_addr + ks * 32);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        if (p.slopes != nullptr) {
          const int row = row0 + rw * 16 + r * 8 + (lane >> 2);
          slope[r] = row < p.G ? p.slopes[kv_head * p.G + row] * 1.4426950408889634f : 0.f;
        }
      }
    }
    // S = Q K^T
    float s[2 * RW][4];
#pragma unroll
    for (int b = 0; b < RW; ++b) {
      float alt[2][4];  // second chain of accumulators: halves the dependent products
#pragma unroll
      for (int e = 0; e < 4; ++e) s[2 * b][e] = s[2 * b + 1][e] = alt[0][e] = alt[1][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t kf[4];
        ldsm4(kf, k_addr + k_line[b] + (ks / 4) * half_stride + (((ks % 4) * 2) ^ k_chunk) * 16);
        if (ks & 1) {
          mma16816<T>(alt[0], qf[ks], kf[0], kf[1]);
          mma16816<T>(alt[1], qf[ks], kf[2], kf[3]);
        } else {
          mma16816<T>(s[2 * b], qf[ks], kf[0], kf[1]);
          mma16816<T>(s[2 * b + 1], qf[ks], kf[2], kf[3]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[2 * b][e] = (s[2 * b][e] + alt[0][e]) * p.scale_log2;
        s[2 * b + 1][e] = (s[2 * b + 1][e] + alt[1][e]) * p.scale_log2;
      }
    }
    const int key_base = t.key0 + kw * RW * 16 + 2 * (lane & 3);
    if (p.slopes != nullptr) {
#pragma unroll
      for (int b = 0; b < 2 * RW; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[b][e] = fmaf(slope[e >> 1], static_cast<float>(key_base + b * 8 + (e & 1) - t.pos), s[b][e]);
    }
    const bool edge = t.key0 < t.lo || t.key0 + kTile > t.hi;
    if (edge) {
#pragma unroll
      for (int b = 0; b < 2 * RW; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key_base + b * 8 + (e & 1);
          if (key < t.lo || key >= t.hi) s[b][e] = -INFINITY;
        }
      // a line outside the keys seen may hold anything (0 * NaN is NaN): clear the V lines this warp reads
#pragma unroll
      for (int b = 0; b < RW; ++b) {
        const int r0 = (kw * RW + b) * 16;
        for (int i = lane; i < 16 * (D / 8); i += 32) {
          const int r = r0 + i / (D / 8), c = i % (D / 8);
          const int key = t.key0 + r;
          if (key < t.lo || key >= t.hi)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_addr + line_offset(r) + (c / 8) * half_stride +
                                                                         (c % 8) * 16),
                         "r"(0)
                         : "memory");
        }
      }
      __syncwarp();
    }
    // running max and rescale
    float base[2];
    bool moved = false;
    float fix[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2 * RW; ++b) mx = fmaxf(mx, fmaxf(s[b][2 * r], s[b][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float next = fmaxf(m[r], mx);
      base[r] = next == -INFINITY ? 0.f : next;
      fix[r] = exp2f(m[r] - base[r]);
      moved |= next != m[r];
      m[r] = next;
      l[r] *= fix[r];
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= fix[0];
        o[i][1] *= fix[0];
        o[i][2] *= fix[1];
        o[i][3] *= fix[1];
      }
    }
    // O += P V
#pragma unroll
    for (int b = 0; b < RW; ++b) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* x = s[2 * b + h];
        x[0] = exp2f(x[0] - base[0]);
        x[1] = exp2f(x[1] - base[0]);
        x[2] = exp2f(x[2] - base[1]);
        x[3] = exp2f(x[3] - base[1]);
        l[0] += x[0] + x[1];
        l[1] += x[2] + x[3];
        split2<T>(x[0], x[1], hi[2 * h], lo[2 * h]);
        split2<T>(x[2], x[3], hi[2 * h + 1], lo[2 * h + 1]);
      }
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) {
        uint32_t vf[4];
        ldsm4_t(vf, v_addr + v_line[b] + (dd / 4) * half_stride + (((dd % 4) * 2) ^ v_chunk) * 16);
        mma16816<T>(o[2 * dd], hi, vf[0], vf[1]);
        mma16816<T>(o[2 * dd + 1], hi, vf[2], vf[3]);
        mma16816<T>(o[2 * dd], lo, vf[0], vf[1]);
        mma16816<T>(o[2 * dd + 1], lo, vf[2], vf[3]);
      }
    }
    if (t.flags & 2) {
      // merge the warps' results through this stage's K and V (4 warps * 16 rows * D floats fill them exactly)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge);  // done with this stage, and with the previous item's s_ml
      if (!mbar_wait_warp(&merge, merge_phase, p.status, kStatusTimeoutAttention, abort_flag)) return;
      merge_phase ^= 1u;
      float* buf = reinterpret_cast<float*>(stages + stage * C::kStageBytes);
      const int rows_live = min(C::kRows, p.G - row0);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = r * 8 + (lane >> 2);
        if ((lane & 3) == 0) s_ml[warp][row] = make_float2(m[r], l[r]);
        if (rw * 16 + row < rows_live) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(buf + (warp * 16 + row) * D + ((i * 8 + 2 * (lane & 3)) ^ ((row & 7) * 8))) =
                make_float2(o[i][2 * r], o[i][2 * r + 1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge);
      if (!mbar_wait_warp(&merge, merge_phase, p.status, kStatusTimeoutAttention, abort_flag)) return;
      merge_phase ^= 1u;
      for (int i = tid; i < rows_live * (D / 4); i += 32 * kWarps) {
        const int row = i / (D / 4), c = (i % (D / 4)) * 4;
        const int rg = row / 16, rr = row % 16;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps / RW; ++w) M = fmaxf(M, s_ml[w * RW + rg][rr].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps / RW; ++w) {
          const float2 ml = s_ml[w * RW + rg][rr];
          const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
          const float4 y = *reinterpret_cast<const float4*>(buf + ((w * RW + rg) * 16 + rr) * D + (c ^ ((rr & 7) * 8)));
          L = fmaf(ml.y, f, L);
          x.x = fmaf(y.x, f, x.x);
          x.y = fmaf(y.y, f, x.y);
          x.z = fmaf(y.z, f, x.z);
          x.w = fmaf(y.w, f, x.w);
        }
        if (t.out < 0) {
          const float inv = 1.f / L;
          T* dst = static_cast<T*>(p.o) + (static_cast<long long>(t.query) * p.Hq + kv_head * p.G + row0 + row) * D + c;
          T y[4] = {from_f32<T>(x.x * inv), from_f32<T>(x.y * inv), from_f32<T>(x.z * inv), from_f32<T>(x.w * inv)};
          *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
        } else {
          const long long at = static_cast<long long>(t.out) * p.part_rows + row;
          *reinterpret_cast<float4*>(p.part_o + at * D + c) = x;
          if (c == 0) p.part_ml[at] = make_float2(M, L);
        }
      }
      __syncwarp();
    }
    // plain stores to the stage come before the next copy into it
    if (edge || (t.flags & 2)) fence_proxy_async_smem();
    if (lane == 0) mbar_arrive(&empty[stage]);
    if (++stage == C::kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
}

// Joins the partials of the item that CTA blockIdx.x began and did not finish: partial 0 in slot 2c + 1, the
// following CTAs' in slot 2c'. Warps take (row, every S-th partial); the S sums of a row are added in order.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(AttnParams p) {
  constexpr int E = D / 32;
  constexpr int kJoinWarps = kJoinThreads / 32;
  __shared__ float s_x[kJoinWarps][D];
  __shared__ float2 s_ml[kJoinWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 join = p.joins[blockIdx.x];
  if (join.w == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kv_head = join.y / p.groups, row0 = (join.y - kv_head * p.groups) * p.part_rows;
  const int rows = min(p.part_rows, p.G - row0);
  int together = 1;  // rows in flight: a power of two up to the warps
  while (together < rows && together < kJoinWarps) together *= 2;
  const int splits = kJoinWarps / together;
  const int slot0 = warp / together;
  for (int r0 = 0; r0 < rows; r0 += together) {
    const int row = r0 + warp % together;
    float M = -INFINITY, L = 0.f, x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
    if (row < rows) {
#pragma unroll 4
      for (int i = slot0; i < join.w; i += splits) {
        const long long at = static_cast<long long>(i == 0 ? 2 * join.z + 1 : 2 * (join.z + i)) * p.part_rows + row;
        const float2 ml = p.part_ml[at];
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = p.part_o[at * D + e * 32 + lane];
        const float next = fmaxf(M, ml.x), base = next == -INFINITY ? 0.f : next;
        const float f = exp2f(M - base), g = exp2f(ml.x - base);
        M = next;
        L = L * f + ml.y * g;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fmaf(y[e], g, x[e] * f);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_x[warp][e * 32 + lane] = x[e];
    if (lane == 0) s_ml[warp] = make_float2(M, L);
    __syncthreads();
    if (warp < together && row < rows) {
      float top = -INFINITY, sum = 0.f, y[E];
      for (int s = 0; s < splits; ++s) top = fmaxf(top, s_ml[s * together + warp].x);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = 0.f;
      for (int s = 0; s < splits; ++s) {
        const float2 ml = s_ml[s * together + warp];
        const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = fmaf(s_x[s * together + warp][e * 32 + lane], f, y[e]);
      }
      T* dst = static_cast<T*>(p.o) + (static_cast<long long>(join.x) * p.Hq + kv_head * p.G + row0 + row) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) dst[e * 32 + lane] = from_f32<T>(y[e] / sum);
    }
    __syncthreads();
  }
}

CUtensorMap page_map(const at::Tensor& t, int dtype) {
  // {64 columns, lines, D / 64 column parts, heads, pages}: one box is a page's lines of one head as
  // D / 64 parts of 128-byte rows
  const uint64_t D = t.size(3), lines = t.size(2);
  const uint64_t dims[5] = {64, lines, D / 64, static_cast<uint64_t>(t.size(1)), static_cast<uint64_t>(t.size(0))};
  auto stride = [&](int d) { return static_cast<uint64_t>(t.size(d) > 1 ? t.stride(d) : D); };
  const uint64_t strides[4] = {stride(2), 64, stride(1), stride(0)};
  const uint32_t box[5] = {64, static_cast<uint32_t>(std::min<uint64_t>(lines, kTile)), static_cast<uint32_t>(D / 64), 1, 1};
  return make_tmap_5d(t.data_ptr(), dtype, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D, int RW>
void launch_attend(AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& q, bool may_split,
                   cudaStream_t stream) {
  using C = Config<D, RW>;
  const int device = q.device().index();
  const auto kernel = attend_kernel<T, D, RW>;
  check_smem_optin(C::kSmem, device, "paged_attention");
  MINT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  const int grid = num_sms(device) * (C::kTwo ? 2 : 1);
  p.groups = (p.G + C::kRows - 1) / C::kRows;
  p.part_rows = p.groups > 1 ? C::kRows : std::min(p.G, C::kRows);
  const int64_t slots = 2ll * grid * p.part_rows;
  auto ws = at::empty({slots * (D + 2) + 4 * grid}, q.options().dtype(at::kFloat));
  p.part_o = ws.data_ptr<float>();
  p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * D);
  p.joins = reinterpret_cast<int4*>(p.part_o + slots * (D + 2));
  kernel<<<grid, kThreads, C::kSmem, stream>>>(tk, tv, p);
  MINT_CUDA_CHECK(cudaGetLastError());
  count_launch();
  if (!may_split) return;
  // launched while the first kernel still runs; it waits for that kernel's end on the device
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  MINT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p));
  count_launch();
}

template <typename T, int D>
void dispatch_rows(AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& q, bool may_split,
                   cudaStream_t stream) {
  if (p.G <= 16) {
    launch_attend<T, D, 1>(p, tk, tv, q, may_split, stream);
  } else if (p.G <= 32) {
    launch_attend<T, D, 2>(p, tk, tv, q, may_split, stream);
  } else {
    launch_attend<T, D, 4>(p, tk, tv, q, may_split, stream);
  }
}

template <typename T>
void dispatch_dim(AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& q, bool may_split,
                  cudaStream_t stream) {
  if (q.size(2) == 64) {
    dispatch_rows<T, 64>(p, tk, tv, q, may_split, stream);
  } else if (q.size(2) == 128) {
    dispatch_rows<T, 128>(p, tk, tv, q, may_split, stream);
  } else {
    dispatch_rows<T, 256>(p, tk, tv, q, may_split, stream);
  }
}

}  // namespace paged

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& tables,
                           const at::Tensor& positions, const c10::optional<at::Tensor>& rows, int64_t window,
                           const c10::optional<at::Tensor>& slopes, double scale) {
  check_contig(q, "q");
  check_cuda(tables, "block_tables");
  check_contig(positions, "positions");
  const auto dt = q.scalar_type();
  MINT_CHECK(q.dim() == 3 && (dt == at::kBFloat16 || dt == at::kHalf), "paged_attention takes bf16 or fp16 [N, Hq, D]");
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2);
  MINT_CHECK(D == 64 || D == 128 || D == 256, "paged_attention takes heads of 64, 128 or 256");
  MINT_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0, "q must be 16-byte aligned");
  MINT_CHECK(kp.dim() == 4 && kp.size(1) >= 1 && Hq >= 1 && Hq % kp.size(1) == 0,
             "query heads must be a multiple of the KV heads");
  paged::check_pool(kp, "k_pages", dt, kp.size(1), D);
  paged::check_pool(vp, "v_pages", dt, kp.size(1), D);
  MINT_CHECK(kp.sizes() == vp.sizes(), "k_pages and v_pages have different shapes");
  MINT_CHECK(tables.dim() == 2 && tables.scalar_type() == at::kInt && (tables.size(1) <= 1 || tables.stride(1) == 1),
             "block_tables must be int32 [B, W] with contiguous rows");
  MINT_CHECK(positions.scalar_type() == at::kInt && positions.numel() == N, "positions are int32, one per query");
  for (const at::Tensor* t : {&kp, &vp, &tables, &positions})
    MINT_CHECK(t->device() == q.device(), "paged_attention takes tensors on one device");
  paged::AttnParams p{};
  if (rows.has_value()) {
    check_contig(*rows, "rows");
    MINT_CHECK(rows->scalar_type() == at::kInt && rows->numel() == N && rows->device() == q.device(),
               "rows are int32, one per query");
    p.rows = rows->data_ptr<int>();
  } else {
    MINT_CHECK(tables.size(0) == N, "without rows there is one table row per query");
  }
  if (slopes.has_value()) {
    check_contig(*slopes, "alibi_slopes");
    MINT_CHECK(slopes->scalar_type() == at::kFloat && slopes->numel() == Hq && slopes->device() == q.device(),
               "alibi_slopes are fp32, one per query head");
    p.slopes = slopes->data_ptr<float>();
  }
  auto o = at::empty_like(q);
  if (N == 0) return o;
  const int shift = paged::shift_of(kp.size(2));
  MINT_CHECK(N < (1 << 24) && Hq < (1 << 16) && tables.size(0) < (1ll << 31) && tables.size(1) <= (INT_MAX >> shift),
             "paged_attention sizes");
  c10::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  p.q = q.data_ptr();
  p.o = o.data_ptr();
  p.tables = tables.data_ptr<int>();
  p.positions = positions.data_ptr<int>();
  p.status = status_ptr(q.device().index());
  p.tstride = tables.stride(0);
  p.N = static_cast<int>(N);
  p.B = static_cast<int>(tables.size(0));
  p.W = static_cast<int>(tables.size(1));
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(kp.size(1));
  p.G = p.Hq / p.Hkv;
  p.n_pages = static_cast<int>(kp.size(0));
  p.page_shift = shift;
  p.window = static_cast<int>(std::max<int64_t>(-1, std::min<int64_t>(window, INT_MAX)));
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  const int type = dt == at::kBFloat16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMap tk = paged::page_map(kp, type), tv = paged::page_map(vp, type);
  // one tile at most per item: nothing to join
  const bool may_split = tables.size(1) * kp.size(2) > paged::kTile;
  if (dt == at::kBFloat16) {
    paged::dispatch_dim<__nv_bfloat16>(p, tk, tv, q, may_split, stream);
  } else {
    paged::dispatch_dim<__half>(p, tk, tv, q, may_split, stream);
  }
  return o;
}

}  // namespace mint
