// Attention of single query tokens over a paged key-value cache.
//
// Query i (position pos of request row) sees keys j in [max(0, pos - window), pos]:
//   o = sum_j softmax_j(scale * q . k_j - slope_h * (pos - j)) v_j
// K and V are read once each: 4 * D bytes per key and KV head for 4 * D * G flops (the G query heads that
// share a KV head), at most 16 flops per byte for G = 16, so HBM bandwidth is the bound and the design is
// about keeping enough bytes in flight on every SM whatever the lengths are.
//
// * Work is cut into tiles of 64 (or 128) keys of one KV head (item = query x KV head). The kernel computes, from the
//   positions on the device, how many tiles there are and gives every CTA an equal contiguous share, so one
//   request of any length, or a batch of mixed lengths, fills the GPU without a plan from the host (and a
//   CUDA graph follows the lengths). A CTA whose share starts or ends inside an item leaves an fp32 partial
//   (running max, sum, unnormalized output); a second, small kernel joins an item's partials in tile order,
//   so results do not depend on timing.
// * Two producer warps, one for K and one for V (a thread issues a box every ~90 cycles, and a tile has 8 boxes
//   of 16 lines each), read the block table 32 entries at a time and issue one TMA box per page (128-byte
//   swizzle, so the fragment loads are free of bank conflicts) into a ring of stages. Pages that hold no
//   visible key are requested out of range: TMA fills zeros and reads nothing, and a corrupt table entry
//   cannot read outside the pool.
// * Four consumer warps take 16 (32) keys of a tile each and keep their own running max, sum and output in
//   registers, so there is no exchange until an item ends, when the warps' results are merged through the
//   item's last stage. Products run on mma.sync m16n8k16 with the keys (S^T = K Q^T) and the output columns
//   (O^T = V^T P^T) on the M side and 8 query rows per N block: a group of 1 to 8 query heads fills one block,
//   where a tcgen05 tile (M = 128 query rows) would be 94 % padding and the tensor pipe is not the bound.
// * Probabilities are split into two 16-bit terms, p = hi + lo, for the second product: they keep 16 bits of
//   precision instead of bf16's 8. fp16 has no exponents for small p: there both p and the running sum are
//   2^15 times the probability relative to the running max, which puts the error of hi + lo below 2^-38 (16 bits
//   for keys down to 15 nats under the max, 11 bits down to 18). Groups of at most 4 heads get the split for
//   nothing: columns 4-7 of the N block repeat the rows, carry lo where columns 0-3 carry hi, and are added when
//   the item ends. Scores, sums and outputs are fp32.
//
// Measured in CUDA graphs: 64 requests of 1024 to 32768 keys (16 heads over 4 of 128, pages of 16, 2.2 GB) 331 us, 6.7 TB/s, the
// rate of a plain copy; the same with 8-line pages 90 % of it. Short work is bound by the chain of dependent reads
// (position, table entry, keys: 0.65 us each), the merge and the join: one tile takes 5.2 us, a ragged batch of
// 44 MB in windows of 512 15.6 us, one request of 131072 keys 51 us (41 us at the copy rate). Two CTAs per SM with
// three 32 KB stages each keep 190 KB in flight.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "paged.cuh"

namespace mint {
namespace paged {

// Keys per tile: 64-wide heads take twice as many, since a tile's latencies do not shrink with its bytes
// (64 requests of 4096 keys, 64 heads over 4, pages of 16: 57.9 us with tiles of 64, 54.4 us with 128).
template <int D>
constexpr int kTileOf = D == 64 ? 128 : 64;
constexpr int kWarps = 4;          // consumer warps
constexpr int kThreads = 32 * (kWarps + 2);  // and a producer warp each for K and V
constexpr int kJoinWarps = 8;

// NB blocks of 8 query rows per item; TWIN: one block whose columns 4-7 repeat rows 0-3 (hi / lo terms)
template <int D, int NB>
struct Config {
  static constexpr int kTile = kTileOf<D>;
  static constexpr int kBlocks = kTile / (16 * kWarps);  // of 16 keys per warp
  static constexpr int kRows = 8 * NB;                   // query rows per item
  static constexpr int kKvBytes = kTile * D * 2;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kStageBytes = (2 * kKvBytes + kQBytes + 1023) / 1024 * 1024;
  static constexpr int kControl = 3072;  // scan, barriers, tile descriptions, merge statistics, base alignment
  static constexpr int kSmSmem = 228 * 1024, kCtaSmem = 227 * 1024;
  static constexpr int fit(int ctas) { return ((ctas > 1 ? kSmSmem / ctas - 1024 : kCtaSmem) - kControl) / kStageBytes; }
  // two CTAs per SM where three stages fit twice, else one
  static constexpr int kCtas = fit(2) >= 3 ? 2 : 1;
  static constexpr int kStages = fit(kCtas) < 6 ? fit(kCtas) : 6;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kMergeLine = D + 4;  // lines of the merge buffer (a stage), padded against bank conflicts
  static_assert(kStages >= 3 || D == 256, "stages");
  static_assert(kStages >= 2 && kSmem + kControl - 1024 <= kCtaSmem, "shared memory");
  static_assert(kWarps * kRows * kMergeLine * 4 <= kStageBytes, "merge buffer");
};

struct alignas(16) TileInfo {  // the tile in a stage, for the consumers
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

// 8x8 transpose of 16-bit elements spread over a warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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

// What probabilities (at most 1) are multiplied by before they are split; it cancels in the division by the sum.
template <typename T>
constexpr float kProbScale = 1.f;
template <>
constexpr float kProbScale<__half> = 32768.f;

// (a, b) = hi + lo in two packed 16-bit pairs: hi is rounded toward zero, so that lo, what that lost, is never
// negative, and neither is below the smallest step of its type's grid (2^-126, or 2^-24 of fp16's 2^15): 0 times an
// infinite value would be NaN, and a lo of the other sign would turn infinity into NaN. The floor adds nothing where
// keys are masked (their values are zeroed) and at most 2^-39 of the largest probability to each term elsewhere.
__device__ __forceinline__ uint32_t at_least(uint32_t x, __nv_bfloat162 least) {
  const __nv_bfloat162 y = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), least);
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t at_least(uint32_t x, __half2 least) {
  const __half2 y = __hmax2_nan(*reinterpret_cast<const __half2*>(&x), least);
  return *reinterpret_cast<const uint32_t*>(&y);
}
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float a, float b, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
  const float2 f = bf16x2_to_float2(hi);
  const __nv_bfloat162 least = __halves2bfloat162(__ushort_as_bfloat16(0x0080), __ushort_as_bfloat16(0x0080));
  lo = at_least(pack_bf16x2(a - f.x, b - f.y), least);
  hi = at_least(hi, least);
}
template <>
__device__ __forceinline__ void split2<__half>(float a, float b, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const __half2 least = __halves2half2(__ushort_as_half(1), __ushort_as_half(1));
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  lo = at_least(*reinterpret_cast<const uint32_t*>(&l), least);
  hi = at_least(hi, least);
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
  template <int TILE>
  __device__ __forceinline__ int tiles() const {
    return hi > 0 ? (hi - 1) / TILE - lo / TILE + 1 : 0;
  }
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

// CTA c of `ctas` owns tiles [share(c), share(c + 1)) of `all`
struct Shares {
  int each, extra;  // the first `extra` CTAs own one tile more
  __device__ __forceinline__ Shares(int all, int ctas) : each(all / ctas), extra(all - all / ctas * ctas) {}
  __device__ __forceinline__ int begin(int c) const { return each * c + min(c, extra); }
  __device__ __forceinline__ int owner(int tile) const {
    const int big = extra * (each + 1);
    return tile < big ? tile / (each + 1) : extra + (tile - big) / each;
  }
};

// mbar_wait_warp that polls a while before it reads the clock and the wait limit (a global load, as long as
// the whole wait for a tile)
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, uint32_t* status, volatile int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  for (int i = 0; i < 64; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(addr, parity))) return true;
  }
  return mbar_wait_warp(bar, parity, status, kStatusTimeoutAttention, abort_flag);
}

template <typename T, int D, int NB, bool TWIN>
__global__ void __launch_bounds__(kThreads, Config<D, NB>::kCtas)
    attend_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, AttnParams p) {
  using C = Config<D, NB>;
  constexpr int kTile = C::kTile, KB = C::kBlocks;
  extern __shared__ uint8_t s_raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages], merge;
  __shared__ TileInfo info[C::kStages];
  __shared__ float2 s_ml[kWarps][C::kRows];
  __shared__ int s_inc[kThreads], s_sum[kThreads / 32], s_abort;
  uint8_t* stages = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x;
  const int per_query = p.Hkv * p.groups;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // this CTA's share of the tiles: totals by a scan over the queries, `chunk` of them per thread
  const int chunk = (p.N + kThreads - 1) / kThreads;
  const int n0 = min(p.N, tid * chunk), n1 = min(p.N, n0 + chunk);
  int inc = 0;
  for (int n = n0; n < n1; ++n) inc += span_at(p, n).template tiles<kTile>();
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 2);
      mbar_init(&empty[i], kWarps);
    }
    mbar_init(&merge, kWarps);
    s_abort = 0;
    fence_mbar_init();
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += up;
  }
  s_inc[tid] = inc;
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += s_sum[w];
  const int all = total * per_query;  // the host keeps it below 2^31
  // shares of one tile if there are few: at least two per CTA took 0.8 us longer for 4 requests of 1000 keys
  const int ctas = max(1, min(static_cast<int>(gridDim.x), all));
  const Shares shares(all, ctas);
  const int t0 = cta < ctas ? shares.begin(cta) : all, t1 = cta < ctas ? shares.begin(cta + 1) : all;
  const int count = t1 - t0;

  if (warp >= kWarps) {
    // ------------------------------------------------------------------------------ producers
    const bool is_k = warp == kWarps;
    int query = 0, off = 0, left = count;
    if (count > 0) {  // the share's first query: the chunk that holds tile t0, then the query in it
      const int u = t0 / per_query;
      int sum = 0, at = 0, owner = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        const int end = sum + s_inc[w * 32 + lane];
        const unsigned past = __ballot_sync(0xffffffffu, end <= u);
        owner += __popc(past);
        if (past != 0) at = __shfl_sync(0xffffffffu, end, 31 - __clz(past));
        sum += s_sum[w];
      }
      query = owner * chunk;
      if (chunk > 1) {
        while (true) {
          int end = query + lane < p.N ? span_at(p, query + lane).template tiles<kTile>() : 0;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end += up;
          }
          end += at;
          const unsigned past = __ballot_sync(0xffffffffu, end <= u);
          if (past != 0) at = __shfl_sync(0xffffffffu, end, 31 - __clz(past));
          query += __popc(past);
          if (past != 0xffffffffu) break;
        }
      }
      off = t0 - at * per_query;
    }
    struct Piece {  // a run of one item's tiles
      Span s;
      int query, group, at, len, tiles;
    };
    auto next_piece = [&]() {
      Piece c{};
      while (left > 0) {
        c.s = span_at(p, query);
        c.tiles = c.s.template tiles<kTile>();
        if (off < c.tiles * per_query) break;
        ++query;
        off = 0;
      }
      if (left > 0) {
        c.query = query;
        c.group = off / c.tiles;
        c.at = off - c.group * c.tiles;
        c.len = min(left, c.tiles - c.at);
        off += c.len;
        left -= c.len;
      }
      return c;
    };
    // 32 table entries at a time, one per lane; entries of the next run are on their way while one is used
    auto entries = [&](const Span& s, int page) {
      return page + lane <= (s.pos >> p.page_shift) ? p.tables[s.row * p.tstride + page + lane] : -1;
    };
    auto first_page = [&](const Piece& c) { return ((c.s.lo / kTile + c.at) * kTile) >> p.page_shift; };
    const int box_lines = min(1 << p.page_shift, kTile), boxes = kTile / box_lines;
    const CUtensorMap* map = is_k ? &tk : &tv;
    int4 join = make_int4(0, 0, 0, 0);
    bool ok = true, bad = false;
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    Piece cur = next_piece();
    int base = 0, entry = -1;
    if (cur.len > 0) {
      base = first_page(cur);
      entry = entries(cur.s, base);
    }
    while (cur.len > 0 && ok) {
      const int rest = left;  // tiles of this CTA after `cur`
      const int kv_head = cur.group / p.groups, row0 = (cur.group - kv_head * p.groups) * C::kRows;
      const int live_rows = min(C::kRows, p.G - row0);
      int out = -1;
      if (cur.at > 0) {
        out = 2 * cta;
      } else if (cur.len < cur.tiles) {
        out = 2 * cta + 1;
        join = make_int4(cur.query, cur.group, cta, shares.owner(t1 - rest - cur.len + cur.tiles - 1) - cta + 1);
      }
      const int last_page = cur.s.pos >> p.page_shift;
      Piece nxt{};
      int ahead = -1, nxt_base = 0, nxt_entry = -1;
      for (int i = 0; i < cur.len; ++i) {
        const int key0 = (cur.s.lo / kTile + cur.at + i) * kTile;
        const int page0 = key0 >> p.page_shift, line = key0 & ((1 << p.page_shift) - 1) & -box_lines;
        if (page0 >= base + 32) {
          base = page0;
          entry = ahead;
          ahead = entries(cur.s, base + 32);
        }
        // a page with no visible key is asked for out of range: zeros, no read
        const int number = base + lane;
        int page = entry;
        if (number > last_page || ((number + 1) << p.page_shift) <= cur.s.lo) {
          page = p.n_pages;
        } else if (page < 0 || page >= p.n_pages) {
          bad = true;
          page = p.n_pages;
        }
        int id[kTile / 8];
#pragma unroll
        for (int b = 0; b < kTile / 8; ++b) id[b] = __shfl_sync(0xffffffffu, page, (page0 - base + b) & 31);
        if (!wait_warp(&empty[stage], phase ^ 1u, p.status, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* buf = stages + stage * C::kStageBytes;
        if (lane == 0) {
          if (is_k)
            info[stage] = TileInfo{cur.query, cur.group, key0, cur.s.lo, cur.s.hi, cur.s.pos, out,
                                   (i == 0 ? 1 : 0) | (i == cur.len - 1 ? 2 : 0)};
          const bool with_q = is_k && i == 0;
          mbar_arrive_expect_tx(&full[stage], C::kKvBytes + (with_q ? live_rows * D * 2 : 0));
          uint8_t* dst = buf + (is_k ? 0 : C::kKvBytes);
#pragma unroll
          for (int b = 0; b < kTile / 8; ++b)
            if (b < boxes) tma_load_page(dst + b * box_lines * D * 2, map, &full[stage], line, kv_head, id[b]);
          if (with_q)
            bulk_load(buf + 2 * C::kKvBytes,
                      static_cast<const T*>(p.q) + (static_cast<long long>(cur.query) * p.Hq + kv_head * p.G + row0) * D,
                      live_rows * D * 2, &full[stage]);
        }
        __syncwarp();
        ++issued;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
        if (i == 0) {  // look ahead once the first copies are out
          ahead = entries(cur.s, base + 32);
          bad |= p.positions[cur.query] != cur.s.pos;
          nxt = next_piece();
          if (nxt.len > 0) {
            nxt_base = first_page(nxt);
            nxt_entry = entries(nxt.s, nxt_base);
          }
        }
      }
      cur = nxt;
      base = nxt_base;
      entry = nxt_entry;
    }
    if (is_k && lane == 0) p.joins[cta] = join;
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
  // tile line r: 64-column parts of a box are half_stride bytes apart, 16-byte chunk c of a line sits at c ^ (r & 7)
  const int box_shift = min(p.page_shift, kTile == 128 ? 7 : 6), box_lines = 1 << box_shift;
  const uint32_t half_stride = box_lines * 128;
  auto line_offset = [&](int r) { return static_cast<uint32_t>((r >> box_shift) * box_lines * D * 2 + (r & (box_lines - 1)) * 128); };
  uint32_t k_line[KB], v_line[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int r0 = (warp * KB + kb) * 16;
    k_line[kb] = line_offset(r0 + (lane & 15));
    v_line[kb] = line_offset(r0 + (lane & 7) + ((lane >> 4) << 3));
  }
  const uint32_t k_chunk = (lane >> 4) ^ (lane & 7), v_chunk = ((lane >> 3) & 1) ^ (lane & 7);
  const uint32_t base_addr = smem_u32(stages);
  const int my_key = warp * KB * 16 + (lane >> 2);  // and + 8, in each block of 16
  const int my_row = 2 * (lane & 3);           // and + 1, in each block of 8

  uint32_t qf[NB][D / 16][2];
  float o[NB][D / 16][4], m[NB][2], l[NB][2], slope[NB][2];
  int stage = 0;
  uint32_t phase = 0, merge_phase = 0;
  for (int it = 0; it < count; ++it) {
    if (!wait_warp(&full[stage], phase, p.status, abort_flag)) return;
    const TileInfo t = info[stage];
    const uint32_t k_addr = base_addr + stage * C::kStageBytes, v_addr = k_addr + C::kKvBytes;
    if (t.flags & 1) {
      const int kv_head = t.group / p.groups, row0 = (t.group - kv_head * p.groups) * C::kRows;
      const int live_rows = min(C::kRows, p.G - row0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        // rows past the last repeat it: they cost nothing and are not written
        const int row = min(TWIN ? lane & 3 : nb * 8 + (lane & 7), live_rows - 1);
        const uint32_t q_addr = k_addr + 2 * C::kKvBytes + row * (D * 2) + (lane >> 3) * 16;
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          uint32_t r[4];
          ldsm4(r, q_addr + ks * 64);
          qf[nb][2 * ks][0] = r[0];
          qf[nb][2 * ks][1] = r[1];
          qf[nb][2 * ks + 1][0] = r[2];
          qf[nb][2 * ks + 1][1] = r[3];
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          m[nb][c] = -INFINITY;
          l[nb][c] = 0.f;
          const int r = min(TWIN ? (my_row + c) & 3 : nb * 8 + my_row + c, live_rows - 1);
          slope[nb][c] = p.slopes != nullptr ? p.slopes[kv_head * p.G + row0 + r] * 1.4426950408889634f : 0.f;
        }
      }
    }
    // S^T = K Q^T: s[kb][nb][0..1] = key my_key, rows my_row, + 1; s[kb][nb][2..3] = key my_key + 8
    float s[KB][NB][4];
    {
      float alt[KB][NB][4];  // second chain of accumulators: halves the dependent products
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[kb][nb][e] = alt[kb][nb][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t kf[4];
          ldsm4(kf, k_addr + k_line[kb] + (ks / 4) * half_stride + (((ks % 4) * 2) ^ k_chunk) * 16);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma16816<T>((ks & 1) ? alt[kb][nb] : s[kb][nb], kf, qf[nb][ks][0], qf[nb][ks][1]);
        }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[kb][nb][e] = (s[kb][nb][e] + alt[kb][nb][e]) * p.scale_log2;
    }
    if (p.slopes != nullptr) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[kb][nb][e] = fmaf(slope[nb][e & 1], static_cast<float>(t.key0 + my_key + kb * 16 + (e >> 1) * 8 - t.pos),
                                s[kb][nb][e]);
    }
    const bool edge = t.key0 < t.lo || t.key0 + kTile > t.hi;
    if (edge) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int key = t.key0 + my_key + kb * 16 + e * 4;
          if (key < t.lo || key >= t.hi) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[kb][nb][e] = s[kb][nb][e + 1] = -INFINITY;
          }
        }
      // a line outside the keys seen may hold anything (0 * NaN is NaN): clear the V lines this warp reads
      for (int i = lane; i < 16 * KB * (D / 8); i += 32) {
        const int r = warp * KB * 16 + i / (D / 8), c = i % (D / 8);
        if (t.key0 + r < t.lo || t.key0 + r >= t.hi)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_addr + line_offset(r) + (c / 8) * half_stride +
                                                                       (c % 8) * 16),
                       "r"(0)
                       : "memory");
      }
      __syncwarp();
    }
    // running max over the keys (lanes 4 apart hold a row's keys) and rescale
    float fix[NB][2];
    bool moved = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = fmaxf(s[0][nb][c], s[0][nb][2 + c]);
#pragma unroll
        for (int kb = 1; kb < KB; ++kb) mx = fmaxf(mx, fmaxf(s[kb][nb][c], s[kb][nb][2 + c]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float next = fmaxf(m[nb][c], mx);
        const float base = next == -INFINITY ? 0.f : next;
        fix[nb][c] = exp2f(m[nb][c] - base);
        moved |= next != m[nb][c];
        m[nb][c] = next;
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          s[kb][nb][c] = exp2f(s[kb][nb][c] - base) * kProbScale<T>;
          s[kb][nb][2 + c] = exp2f(s[kb][nb][2 + c] - base) * kProbScale<T>;
          sum += s[kb][nb][c] + s[kb][nb][2 + c];
        }
        l[nb][c] = fmaf(l[nb][c], fix[nb][c], sum);
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nb][i][e] *= fix[nb][e & 1];
    }
    // O^T += V^T P^T; P^T's operand layout is the transpose of S^T's
    uint32_t hi[KB][NB][2], lo[KB][NB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a, b;
          split2<T>(s[kb][nb][2 * h], s[kb][nb][2 * h + 1], a, b);
          if (TWIN) {
            hi[kb][nb][h] = transpose8((lane & 2) ? b : a);  // columns 4-7 carry lo
          } else {
            hi[kb][nb][h] = transpose8(a);
            lo[kb][nb][h] = transpose8(b);
          }
        }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        uint32_t vf[4];
        ldsm4_t(vf, v_addr + v_line[kb] + (i / 4) * half_stride + (((i % 4) * 2) ^ v_chunk) * 16);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma16816<T>(o[nb][i], vf, hi[kb][nb][0], hi[kb][nb][1]);
          if (!TWIN) mma16816<T>(o[nb][i], vf, lo[kb][nb][0], lo[kb][nb][1]);
        }
      }
    if (t.flags & 2) {
      // merge the warps' results through this stage
      const int kv_head = t.group / p.groups, row0 = (t.group - kv_head * p.groups) * C::kRows;
      const int live_rows = min(C::kRows, p.G - row0);
      float* buf = reinterpret_cast<float*>(stages + stage * C::kStageBytes);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], d);
        }
      if (TWIN) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[0][i][e] += __shfl_xor_sync(0xffffffffu, o[0][i][e], 2);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge);  // done with this stage, and with what was merged before
      if (!wait_warp(&merge, merge_phase, p.status, abort_flag)) return;
      merge_phase ^= 1u;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int row = nb * 8 + my_row + c;
          if (row < live_rows) {
            if (lane < 4) s_ml[warp][row] = make_float2(m[nb][c], l[nb][c]);
            float* dst = buf + (warp * C::kRows + row) * C::kMergeLine + (lane >> 2);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              dst[i * 16] = o[nb][i][c];
              dst[i * 16 + 8] = o[nb][i][2 + c];
            }
          }
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge);
      if (!wait_warp(&merge, merge_phase, p.status, abort_flag)) return;
      merge_phase ^= 1u;
      for (int i = tid; i < live_rows * (D / 4); i += 32 * kWarps) {
        const int row = i / (D / 4), c = (i % (D / 4)) * 4;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_ml[w][row].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = s_ml[w][row];
          const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
          const float4 y = *reinterpret_cast<const float4*>(buf + (w * C::kRows + row) * C::kMergeLine + c);
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
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    if (++stage == C::kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
}

// Joins the partials of the item that CTA blockIdx.x began and did not finish: the first in slot 2c + 1, the
// following CTAs' in slots 2c'. A block takes every gridDim.y-th row (of at most 16); its warps take every 8th
// partial, and the warps' sums are added in order. Bound by its start and two dependent rounds of loads: 1.8 to 3
// us of a call, 6 us when 74 CTAs share an item. Small blocks (32 registers, 2 to 8 KB) fit beside the first
// kernel's CTAs and are waiting when those end; blocks of 512 threads took 2 us longer.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(AttnParams p) {
  constexpr int E = D / 32;
  __shared__ float s_x[kJoinWarps][D];
  __shared__ float2 s_ml[kJoinWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 join = p.joins[blockIdx.x];
  if (join.w == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kv_head = join.y / p.groups, row0 = (join.y - kv_head * p.groups) * p.part_rows;
  const int rows = min(p.part_rows, p.G - row0);
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    float M = -INFINITY, L = 0.f, x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll 4
    for (int i = warp; i < join.w; i += kJoinWarps) {
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
#pragma unroll
    for (int e = 0; e < E; ++e) s_x[warp][e * 32 + lane] = x[e];
    if (lane == 0) s_ml[warp] = make_float2(M, L);
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
      float top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_ml[w].x);
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float2 ml = s_ml[w];
        const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
        sum = fmaf(ml.y, f, sum);
        y = fmaf(s_x[w][d], f, y);
      }
      static_cast<T*>(p.o)[(static_cast<long long>(join.x) * p.Hq + kv_head * p.G + row0 + row) * D + d] =
          from_f32<T>(y / sum);
    }
    __syncthreads();
  }
}

CUtensorMap page_map(const at::Tensor& t, int dtype, int tile) {
  // {64 columns, lines, D / 64 column parts, heads, pages}: one box is a page's lines of one head as
  // D / 64 parts of 128-byte rows
  const uint64_t D = t.size(3), lines = t.size(2);
  const uint64_t dims[5] = {64, lines, D / 64, static_cast<uint64_t>(t.size(1)), static_cast<uint64_t>(t.size(0))};
  auto stride = [&](int d) { return static_cast<uint64_t>(t.size(d) > 1 ? t.stride(d) : D); };
  const uint64_t strides[4] = {stride(2), 64, stride(1), stride(0)};
  const uint32_t box[5] = {64, static_cast<uint32_t>(std::min<uint64_t>(lines, tile)), static_cast<uint32_t>(D / 64), 1, 1};
  return make_tmap_5d(t.data_ptr(), dtype, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D, int NB, bool TWIN>
void launch_attend(AttnParams p, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& q, bool may_split,
                   int64_t tiles_bound, cudaStream_t stream) {
  using C = Config<D, NB>;
  const int device = q.device().index();
  const auto kernel = attend_kernel<T, D, NB, TWIN>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised for this kernel
  if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
    check_smem_optin(C::kSmem, device, "paged_attention");
    MINT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    ready.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  const int grid = num_sms(device) * C::kCtas;
  p.groups = (p.G + C::kRows - 1) / C::kRows;
  p.part_rows = p.groups > 1 ? C::kRows : p.G;
  const int64_t slots = 2ll * grid * p.part_rows;
  auto ws = empty_cuda({may_split ? slots * (D + 2) + 4 * grid : 4 * grid}, at::kFloat, q.device());
  p.joins = reinterpret_cast<int4*>(ws.data_ptr<float>());
  p.part_o = ws.data_ptr<float>() + 4 * grid;
  p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * D);
  // tile numbers are ints: so many queries that they might not fit go in several launches
  const int64_t per_query = tiles_bound * p.Hkv * p.groups;
  MINT_CHECK(per_query <= INT_MAX, "paged_attention: a query may have too many tiles");
  const int step = static_cast<int>(std::min<int64_t>(p.N, INT_MAX / per_query));
  const AttnParams all = p;
  for (int n = 0; n < all.N; n += step) {
    p.N = std::min(step, all.N - n);
    p.q = static_cast<const T*>(all.q) + static_cast<int64_t>(n) * p.Hq * D;
    p.o = static_cast<T*>(all.o) + static_cast<int64_t>(n) * p.Hq * D;
    p.positions = all.positions + n;
    if (all.rows != nullptr) {
      p.rows = all.rows + n;
    } else {
      p.tables = all.tables + n * all.tstride;
      p.B = p.N;
    }
    kernel<<<grid, kThreads, C::kSmem, stream>>>(tk, tv, p);
    MINT_CUDA_CHECK(cudaGetLastError());
    count_launch();
    if (!may_split) continue;
    // launched while the first kernel still runs; it waits for that kernel's end on the device
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, std::min(p.part_rows, 16));
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    MINT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p));
    count_launch();
  }
}

// Query rows per item: 4 (hi and lo terms side by side in one block of 8), 8 or 16. Wider groups are several
// items, which read K and V again (from L2 as far as it holds them): 32 rows at once leave registers for one
// CTA per SM only and measured the same (256 requests of 4096 keys, 32 heads over 1: 204 us against 195).
template <typename T, int D, typename... Args>
void dispatch_rows(const AttnParams& p, Args&&... args) {
  if (p.G <= 4) {
    launch_attend<T, D, 1, true>(p, args...);
  } else if (p.G <= 8) {
    launch_attend<T, D, 1, false>(p, args...);
  } else {
    launch_attend<T, D, 2, false>(p, args...);
  }
}

template <typename T, typename... Args>
void dispatch_dim(const AttnParams& p, int64_t D, Args&&... args) {
  if (D == 64) {
    dispatch_rows<T, 64>(p, args...);
  } else if (D == 128) {
    dispatch_rows<T, 128>(p, args...);
  } else {
    dispatch_rows<T, 256>(p, args...);
  }
}

}  // namespace paged

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& tables,
                           const at::Tensor& positions, const c10::optional<at::Tensor>& rows, int64_t window,
                           const c10::optional<at::Tensor>& slopes, double scale) {
  paged::check_inference("paged_attention", {&q, &kp, &vp});
  if (slopes.has_value()) paged::check_inference("paged_attention", {&*slopes});
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
  auto o = paged::empty_cuda(q.sizes(), dt, q.device());
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
  const int tile = D == 64 ? paged::kTileOf<64> : D == 128 ? paged::kTileOf<128> : paged::kTileOf<256>;
  const CUtensorMap tk = paged::page_map(kp, type, tile), tv = paged::page_map(vp, type, tile);
  // the most tiles that a query can have; with one at most there is nothing to join
  int64_t tiles_bound = std::max<int64_t>(1, (tables.size(1) * kp.size(2) + tile - 1) / tile);
  if (window >= 0) tiles_bound = std::min<int64_t>(tiles_bound, window / tile + 2);
  const bool may_split = tiles_bound > 1;
  if (dt == at::kBFloat16) {
    paged::dispatch_dim<__nv_bfloat16>(p, D, tk, tv, q, may_split, tiles_bound, stream);
  } else {
    paged::dispatch_dim<__half>(p, D, tk, tv, q, may_split, tiles_bound, stream);
  }
  return o;
}

}  // namespace mint
