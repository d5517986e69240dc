// Causal attention of pieces of prompts over the 4-bit cache (format: kv_q4.cuh), for pages of 16
// tokens, head_dim 64 or 128 and at most 128 query heads per KV head; other shapes run on kv_q4.cu's
// one-warp kernel.
//
// Mathematics: softmax(scale q K^T) V with an online softmax over 64 keys at a time, as
// chunk_attention computes it: S = Q K^T and O += P V on tcgen05, O in tensor memory, rescaled only
// when a row's maximum grew by more than 2^8; P is rounded to f16 for the second product (as
// chunk_attention and prefill_attention round it; its relative error, 2^-11 at most and independent
// from key to key, adds to the result about what the result's own rounding to f16 does), its sum is
// kept in f32. The largest weight is 2^7 to 2^15, so that relative error holds for weights down to 2^-21
// of it; smaller ones are off by up to 2^-32 of it. K and V enter as f16 tiles; every value of the cache is an f16 number, so unpacking
// rounds nothing.
//
// Roles of a CTA's sixteen warps: warp 0 brings Q (TMA) and the pages' 4-bit records (bulk copies);
// warps 1 and 2 issue the MMAs, one for each tile; warps 4-7 unpack a 128-key tile of K or V into the 128-byte-swizzled layout
// the tensor cores read; warps 8-15 are two softmax warpgroups, one query row per thread.
//
// Rows. The M = 128 rows of a tile are (token, query head) pairs of ONE KV head: 128 / hq tokens times
// its hq heads. So a KV head's keys are unpacked once for all heads that share it, and a piece of a
// few tokens still fills a tile hq times better than a tile per head would.
//
// Work split. A unit is (piece, KV head, block of two tiles); its work is the 128-key tiles its last
// row sees. The units' tiles form one list, a CTA takes an equal, contiguous share of it (one CTA per
// SM), whatever the pieces' lengths are. A unit that is cut leaves one partial in each CTA (f32
// numerator, maximum and sum), which a second kernel joins. A block that fits one tile (a piece of a
// few rows) is worked on by both: they hold the same rows, one takes the first 64 keys of every 128,
// the other the second, and their results are joined at the end. (One softmax warpgroup alone waits
// for its own latencies: 1.9 us per 128 keys against 1.25 us for two of them.)
//
// Bound: the tensor cores by operations; measured, the softmax warps (1700 of 1870 cycles per 64 keys, 1024 of them
// the exponentials' unit) with the unpacking in the same issue slots. 2048 rows at position 30000, 32/8 heads, D 128:
// 888 us at 1965 MHz, 1170 TFLOP/s; 1023-1034 us at the 1695 MHz that the power cap leaves. 8 pieces of 1-8 rows at
// 700-6000: 39 us, where unpacking a tile (1650 cycles) sets the pace.
//
// NaN. A weight of zero times a NaN is a NaN, so a spoilt V row would reach rows that do not see it.
// The unpacking warps store zeros for it instead and note the least such position of each 64-column
// group; a row at or behind it gets its NaN at the end.
#include "kv_q4.cuh"

namespace tb {

namespace {

constexpr int CQ_BM = 128;       // rows of a tile
constexpr int CQ_BN = 128;       // keys of a K / V tile
constexpr int CQ_SN = 64;        // keys of a sub-block: the unit of S, softmax and P V
constexpr int CQ_THREADS = 512;  // warps 0 TMA, 1-2 MMA, (3 idle), 4-7 unpack, 8-15 softmax
constexpr int CQ_LEAST = 1;      // tiles a CTA takes at least
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f;
constexpr float P_AIM = 7.0f;  // log2 of a row's largest weight when its reference is set: up to 2^15 later, an f16 holds 2^16

// What a table entry outside the cache reads as.
__device__ __align__(128) unsigned char g_zero_record[2048];

struct CqParams {
  const unsigned char* Kc;
  const unsigned char* Vc;
  const int* table;
  const int* meta;
  __half* O;
  float* part;  // [CTA][2][D + 2][256]: a row's numerator, maximum and sum, rows side by side
  int* desc;    // [CTA][4]: piece, KV head, block, CTAs that hold a part of the unit cut at this CTA's end (0: none)
  float scale;
  int T, H, G, hq, tm, C, NP, MP;  // tm: tokens of a tile
  unsigned int* status;
};

template <int D>
struct CqSmem {
  static constexpr int SUB = D / 64;
  static constexpr int REC = 16 * (D / 2 + 2 * SUB);
  static constexpr int Q_TILE = CQ_BM * D * 2;
  static constexpr int KV_BYTES = CQ_BN * D * 2;
  static constexpr int RAW = 8 * REC;  // a tile's records
  static constexpr int NSLOT = 4;
  static constexpr int NRAW = D == 128 ? 3 : 4;
  static constexpr int OFF_KV = 2 * Q_TILE;
  static constexpr int OFF_RAW = OFF_KV + NSLOT * KV_BYTES;
  static constexpr int OFF_BAR = OFF_RAW + NRAW * RAW;
  static constexpr int OFF_EX = OFF_BAR + 40 * 8;  // a narrow unit's maxima [2][128] and sums [128]
  static constexpr int TOTAL = OFF_EX + 3 * 128 * 4 + 1024;
  static constexpr int TMEM_COLS = 512;
  static_assert(TOTAL <= 227 * 1024, "shared memory");
  static_assert(RAW % 128 == 0 && OFF_BAR % 8 == 0, "alignment");
  static_assert((CQ_THREADS + 8) * 8 <= KV_BYTES, "the prefix sums use the first K / V slot");
};

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// A piece of the step, empty if its descriptor does not lie inside it.
struct Piece {
  int row0, nrows, pos0, blocks;
};
__device__ __forceinline__ Piece piece_of(const CqParams& p, int c) {
  const int4 m = *reinterpret_cast<const int4*>(p.meta + 4 * c);
  Piece r = {m.x, m.y, m.z, 0};
  if (r.row0 < 0 || r.nrows <= 0 || r.pos0 < 0 || r.nrows > p.T - r.row0 || r.nrows > 0x7fffffff - 256 - r.pos0)
    r.nrows = 0;
  r.blocks = (r.nrows + 2 * p.tm - 1) / (2 * p.tm);
  return r;
}
// Tiles of keys that block `i` of a piece sees.
__device__ __forceinline__ int tiles_of(const CqParams& p, const Piece& r, int i) {
  return (r.pos0 + min((i + 1) * 2 * p.tm, r.nrows) + CQ_BN - 1) / CQ_BN;
}

// Walks a CTA's share of the list: `k0`, `k1` are the tiles of the current unit that are its own.
struct Walk {
  int c, g, i, left, share;
  Piece r;
  int tiles, k0, k1;
  bool narrow;  // the block's rows fit one tile

  __device__ __forceinline__ void set(const CqParams& p, int from) {
    tiles = tiles_of(p, r, i);
    narrow = r.nrows - i * 2 * p.tm <= p.tm;
    k0 = from;
    k1 = left < tiles - from ? from + left : tiles;
    left -= k1 - k0;
  }
  // To the next unit; false at the end of the share.
  __device__ __forceinline__ bool next(const CqParams& p) {
    if (left <= 0) return false;
    if (++i == r.blocks) {
      i = 0;
      if (++g == p.G) {
        g = 0;
        do r = piece_of(p, ++c);
        while (r.blocks == 0);  // `left` says that one follows
      }
    }
    set(p, 0);
    return true;
  }
};

// Where this CTA begins. All threads call it. False: it has no share.
__device__ __forceinline__ bool find_walk(const CqParams& p, long long* scan, Walk* w) {
  const int per = (p.C + CQ_THREADS - 1) / CQ_THREADS;
  const int c0 = min(p.C, (int)threadIdx.x * per), c1 = min(p.C, c0 + per);
  auto tiles_in = [&](int c) {
    const Piece r = piece_of(p, c);
    long long s = 0;
    for (int i = 0; i < r.blocks; ++i) s += tiles_of(p, r, i);
    return s;
  };
  long long sum = 0;
  for (int c = c0; c < c1; ++c) sum += tiles_in(c);
  scan[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    constexpr int OWN = CQ_THREADS / 32;
    long long own = 0;
    for (int i = 0; i < OWN; ++i) own += scan[threadIdx.x * OWN + i];
    long long inc = own;
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if ((int)threadIdx.x >= o) inc += up;
    }
    long long at = inc - own;
    for (int i = 0; i < OWN; ++i) {
      const long long v = scan[threadIdx.x * OWN + i];
      scan[threadIdx.x * OWN + i] = at;
      at += v;
    }
    if (threadIdx.x == 31) scan[CQ_THREADS] = at;
  }
  __syncthreads();
  const long long all = scan[CQ_THREADS] * p.G;
  const long long share = max((all + gridDim.x - 1) / gridDim.x, (long long)CQ_LEAST);
  const long long start = blockIdx.x * share;
  if (start >= all) return false;  // uniform for the CTA
  long long at = scan[threadIdx.x] * p.G;
  for (int c = c0; c < c1; ++c) {
    const long long n = tiles_in(c);
    if (start >= at && start < at + n * p.G) {
      const Piece r = piece_of(p, c);
      long long in = (start - at) % n;
      int i = 0;
      for (; in >= tiles_of(p, r, i); ++i) in -= tiles_of(p, r, i);
      scan[CQ_THREADS + 1] = c, scan[CQ_THREADS + 2] = (start - at) / n, scan[CQ_THREADS + 3] = i, scan[CQ_THREADS + 4] = in;
    }
    at += n * p.G;
  }
  __syncthreads();
  w->c = (int)scan[CQ_THREADS + 1], w->g = (int)scan[CQ_THREADS + 2], w->i = (int)scan[CQ_THREADS + 3];
  w->share = (int)share;  // (2^31 tiles would be hours of work)
  w->left = (int)min(share, all - start);
  w->r = piece_of(p, w->c);
  w->set(p, (int)scan[CQ_THREADS + 4]);
  return true;
}

// Sub-blocks of keys that tile `t` of the current unit visits in this CTA's part. In a narrow unit
// sub-block n of tile t is half t of K / V tile n, else half n & 1 of tile n >> 1.
__device__ __forceinline__ int subs_of(const CqParams& p, const Walk& w, int t) {
  const int first = w.i * 2 * p.tm + (w.narrow ? 0 : t * p.tm);
  if (first >= w.r.nrows) return 0;
  const int end = min(CQ_BN * w.k1, w.r.pos0 + min(first + p.tm, w.r.nrows));
  const int subs = max(0, (end - CQ_BN * w.k0 + CQ_SN - 1) / CQ_SN);
  return w.narrow ? (subs + 1 - t) / 2 : subs;
}

template <int D>
__global__ void __launch_bounds__(CQ_THREADS, 1) chunk_q4_kernel(const __grid_constant__ CUtensorMap mapQ, const CqParams p) {
  using SM = CqSmem<D>;
  constexpr int SUB = SM::SUB, NSLOT = SM::NSLOT, NRAW = SM::NRAW;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + SM::OFF_BAR);
  uint64_t* q_full = bars;              // a unit's Q has landed
  uint64_t* q_free = bars + 1;          // and each tile's last S has been computed
  uint64_t* raw_full = bars + 2;        // [NRAW]
  uint64_t* raw_empty = bars + 6;       // [NRAW]
  uint64_t* kv_full = bars + 10;        // [NSLOT]
  uint64_t* kv_empty = bars + 14;       // [NSLOT]
  uint64_t* s_full = bars + 18;         // [tile][buffer]
  uint64_t* p_ready = bars + 22;        // [tile][buffer]
  uint64_t* o_done = bars + 26;         // [tile][parity]
  uint32_t* tmem_slot = (uint32_t*)(bars + 30);
  int* nan_at = (int*)(bars + 31);      // [unit & 7][group]: least position of a spoilt V row

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_free, 2);
    for (int i = 0; i < NRAW; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    for (int i = 0; i < NSLOT; ++i) {
      mbar_init(&kv_full[i], 128);
      mbar_init(&kv_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], CQ_BM);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 16; ++i) nan_at[i] = 0x7fffffff;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, SM::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  pdl_wait();
  if (threadIdx.x == 0) p.desc[4 * blockIdx.x + 3] = 0;
  Walk w;
  const bool busy = find_walk(p, (long long*)(smem + SM::OFF_KV), &w);
  __syncthreads();  // the prefix sums lie where the first tile will
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (!busy) {
    // Nothing to do but to give the tensor memory back.
  } else if (warp < 4) {
    if (warp == 0) {
      // ---- Q and the records of K and V tiles, in the order K V K V ... -----------------------------
      if (lane == 0) prefetch_tmap(&mapQ);
      int item = 0, unit = 0;
      do {
        const int slim = w.r.pos0 + w.r.nrows;
        // Lane j < 8: the page of keys [128 k + 16 j, + 16). Beyond the table: page 0; behind the last key,
        // or outside the cache: zeros. Looked up a tile ahead.
        auto page_of = [&](int k) {
          const int col = k * 8 + (lane & 7);
          return k >= w.k1 || (long long)col * 16 >= slim ? -1 : col < p.MP ? p.table[(size_t)w.r.row0 * p.MP + col] : 0;
        };
        auto load_q = [&]() {
          if (lane == 0) {
            mbar_expect_tx(q_full, 2 * SUB * p.tm * p.hq * 128);
            const int row = w.r.row0 + w.i * 2 * p.tm;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int sub = 0; sub < SUB; ++sub)
                tma_load_3d(smem + t * SM::Q_TILE + sub * (CQ_BM * 128), &mapQ, q_full, sub * 64, w.g * p.hq, row + (w.narrow ? 0 : t * p.tm));
          }
          __syncwarp();
        };
        int next = page_of(w.k0);
        if (unit == 0) load_q();
        for (int k = w.k0; k < w.k1; ++k) {
          const int page = next;
          next = page_of(k + 1);
          const bool in = page >= 0 && page < p.NP;
          const size_t off = ((size_t)(in ? page : 0) * p.G + w.g) * SM::REC;
#pragma unroll
          for (int v = 0; v < 2; ++v, ++item) {
            const int s = item % NRAW;
            if (lane == 0) {
              if (item >= NRAW) mbar_wait(&raw_empty[s], (item / NRAW - 1) & 1, p.status, 602);
              mbar_expect_tx(&raw_full[s], SM::RAW);
            }
            __syncwarp();
            if (lane < 8)
              bulk_load(smem + SM::OFF_RAW + s * SM::RAW + lane * SM::REC, in ? (v ? p.Vc : p.Kc) + off : g_zero_record, SM::REC,
                        &raw_full[s]);
          }
          // Behind the first tile's records: the unpacking warps fetch a unit's first tile before they convert
          // the last one of the unit before, whose products free Q's place.
          if (k == w.k0 && unit > 0) {
            if (lane == 0) mbar_wait(q_free, (unit - 1) & 1, p.status, 601);
            load_q();
          }
        }
        ++unit;
      } while (w.next(p));
    } else if (warp < 3 && elect_one()) {
      // ---- MMA issue: a warp per tile -----------------------------------------------------------------
      // (One thread issuing for both was the kernel's clock: with its waits and fences it took 2240 cycles
      // for a sub-block of both tiles, whose products take 1024.)
      constexpr uint32_t idesc_s = umma_idesc_f16(CQ_BM, CQ_SN, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc_f16(CQ_BM, D, 0, 1);
      const int t = warp - 1;
      const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * D;
      const uint64_t qd = umma_desc_sw128(smem_u32(smem + t * SM::Q_TILE), 16, 1024);
      int base = 0, done = 0;   // K and V tiles, and this tile's sub-blocks, of earlier units: buffers and phases follow
      int ready = 0, unit = 0;  // tiles [0, ready) have been unpacked
      auto slot_addr = [&](int item) { return smem_u32(smem + SM::OFF_KV + (item % NSLOT) * SM::KV_BYTES); };
      auto need = [&](int item) {
        if (ready > item) return;
        while (ready <= item) {
          mbar_wait(&kv_full[ready % NSLOT], (ready / NSLOT) & 1, p.status, 603);
          ++ready;
        }
        tc_fence_after();
      };
      do {
        const int nt = subs_of(p, w, t), nitems = 2 * (w.k1 - w.k0);
        // Sub-block n's K (V) tile, its half of it, and whether it is the tile's last sub-block.
        auto tile_of = [&](int n) { return w.narrow ? n : n >> 1; };
        auto half_of = [&](int n) { return w.narrow ? t : n & 1; };
        auto last_of = [&](int n) { return w.narrow || (n & 1); };
        // (Descriptors hold addresses in units of 16 bytes.)
        auto issue_s = [&](int n) {
          const int b = (done + n) & 1;
          const uint64_t kd0 = umma_desc_sw128(slot_addr(base + 2 * tile_of(n)) + half_of(n) * (CQ_SN * 128), 16, 1024);
#pragma unroll
          for (int kd = 0; kd < D / 16; ++kd) {
            const uint32_t off = ((kd >> 2) * (CQ_BM * 128) + (kd & 3) * 32) >> 4;
            umma_f16(ts + b * CQ_SN, qd + off, kd0 + off, idesc_s, kd > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[t * 2 + b]);
        };
        auto issue_pv = [&](int n) {
          const int b = (done + n) & 1;
          const uint64_t vd = umma_desc_sw128(slot_addr(base + 2 * tile_of(n) + 1) + half_of(n) * (CQ_SN * 128), CQ_BN * 128, 1024);
#pragma unroll
          for (int kk = 0; kk < CQ_SN / 16; ++kk)
            umma_f16_ts(to, ts + b * CQ_SN + kk * 8, vd + kk * (2048 >> 4), idesc_o, (n > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&o_done[t * 2 + b]);
        };
        mbar_wait(q_full, unit & 1, p.status, 604);
        tc_fence_after();
        // A K or V tile is given back once its products are issued; those that no sub-block of this tile
        // reads (a last one's second half, keys behind its rows) at the end.
        int freed_k = 0, freed_v = 0;
        if (nt == 0) umma_commit(q_free);
        for (int n = 0; n < 2 && n < nt; ++n) {
          need(base + 2 * tile_of(n));
          issue_s(n);
          if (n + 1 == nt) umma_commit(q_free);
          if (last_of(n)) umma_commit(&kv_empty[(base + 2 * freed_k++) % NSLOT]);
        }
        for (int n = 0; n < nt; ++n) {
          const int b = done + n;
          need(base + 2 * tile_of(n) + 1);
          mbar_wait(&p_ready[t * 2 + (b & 1)], (b >> 1) & 1, p.status, 605);
          tc_fence_after();
          issue_pv(n);
          if (last_of(n)) umma_commit(&kv_empty[(base + 2 * freed_v++ + 1) % NSLOT]);
          if (n + 2 < nt) {
            need(base + 2 * tile_of(n + 2));
            issue_s(n + 2);
            if (n + 3 == nt) umma_commit(q_free);
            if (last_of(n + 2)) umma_commit(&kv_empty[(base + 2 * freed_k++) % NSLOT]);
          }
        }
        for (; 2 * freed_k < nitems || 2 * freed_v < nitems;) {
          // In the order of the items: a tile can only be given back once it is there.
          const bool k = freed_k <= freed_v && 2 * freed_k < nitems;
          const int item = k ? 2 * freed_k++ : 2 * freed_v++ + 1;
          need(base + item);
          umma_commit(&kv_empty[(base + item) % NSLOT]);
        }
        base += nitems;
        done += nt;
        ++unit;
      } while (w.next(p));
    }
  } else if (warp < 8) {
    // ---- unpack: a thread takes 32 neighbouring elements of a key, of ITER keys a fixed distance apart ----
    // (straight-line code: the loads of all its keys are in flight before the first is used)
    constexpr int PARTS = D / 32;           // 16-byte pieces of a row of codes
    constexpr int STEP = 128 / PARTS;       // keys between a thread's keys
    constexpr int ITER = CQ_BN / STEP;
    static_assert(STEP % 16 == 0, "a thread's keys have one place in their pages");
    const int tid = threadIdx.x - 128, part = tid % PARTS, key0 = tid / PARTS;
    const int from = (key0 >> 4) * SM::REC + (key0 & 15) * (D / 2) + part * 16;
    const int head_from = (key0 >> 4) * SM::REC + 8 * D + 2 * ((key0 & 15) * SUB + (part >> 1));
    // The four 16-byte chunks this thread's words become, in the swizzled tile. Pieces 2 and 3 lie in the
    // other 64-column block, at the same banks: they go in another order.
    uint32_t to[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      to[i] = (part >> 1) * (CQ_BN * 128) + key0 * 128 + (((((part & 1) * 4 + (i ^ (part & 2))) ^ (key0 & 7))) << 4);
    const __half2 R = __float2half2_rn(0.0625f);
    const uint32_t smem_at = smem_u32(smem);
    // `fetch` takes the next item's codes and headers into registers, a step ahead of their conversion, and
    // gives the raw slot back at once. Headers behind the last key are stale and count as zero; spoilt
    // headers of V are noted and count as zero.
    uint4 u[ITER], un[ITER];
    uint32_t head[ITER], headn[ITER];
    int fetched = 0, unit = 0, k = w.k0, v = 0;  // the item that is fetched next, its unit, tile and cache
    bool more = true;
    auto fetch = [&]() {
      const int rs = fetched % NRAW;
      mbar_wait(&raw_full[rs], (fetched / NRAW) & 1, p.status, 606);
      const uint32_t raw = smem_at + SM::OFF_RAW + rs * SM::RAW;
#pragma unroll
      for (int j = 0; j < ITER; ++j) {
        // (Pieces 2 and 3 swap their halves here: see `to`.)
        const uint32_t c = raw + from + j * (STEP / 16) * SM::REC;
        const uint2 lo = lds64(c + (part & 2) * 4), hi = lds64(c + 8 - (part & 2) * 4);
        un[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        headn[j] = lds16(raw + head_from + j * (STEP / 16) * SM::REC);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty[rs]);
      const int slim = w.r.pos0 + w.r.nrows, at = k * CQ_BN + key0;
      if ((k + 1) * CQ_BN > slim) {
#pragma unroll
        for (int j = 0; j < ITER; ++j)
          if (at + j * STEP >= slim) headn[j] = 0;
      }
      if (v) {
        bool spoilt = false;
#pragma unroll
        for (int j = 0; j < ITER; ++j) spoilt |= (headn[j] & 0x7c00u) == 0x7c00u;
        if (spoilt) {
#pragma unroll
          for (int j = 0; j < ITER; ++j)
            if ((headn[j] & 0x7c00u) == 0x7c00u) {
              atomicMin(&nan_at[(unit & 7) * 2 + (part >> 1)], at + j * STEP);
              headn[j] = 0;
            }
        }
      }
      ++fetched;
      v ^= 1;
      if (v == 0 && ++k == w.k1) {
        more = w.next(p);
        k = w.k0;
        ++unit;
      }
    };
    fetch();
    bool have = true;
#pragma unroll 1
    for (int item = 0; have; ++item) {
#pragma unroll
      for (int j = 0; j < ITER; ++j) u[j] = un[j], head[j] = headn[j];
      have = more;
      if (more) fetch();
      const int s = item % NSLOT;
      if (item >= NSLOT) mbar_wait(&kv_empty[s], (item / NSLOT - 1) & 1, p.status, 607);
      const uint32_t dst = smem_at + SM::OFF_KV + s * SM::KV_BYTES;
#pragma unroll
      for (int j = 0; j < ITER; ++j) {
        const uint32_t z = head[j] & 15u;
        // Scale, -(1024 + z) and -(64 + z), twice each.
        const uint32_t sc = __byte_perm(head[j] & 0xfff0u, 0, 0x1010), c0 = (z | z << 16) | 0xe400e400u,
                       c1 = (z << 4 | z << 20) | 0xd400d400u;
        const __half2 S = *reinterpret_cast<const __half2*>(&sc), A = *reinterpret_cast<const __half2*>(&c0), B = *reinterpret_cast<const __half2*>(&c1);
        const uint32_t word[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t up = word[i] >> 8;
          uint32_t e[4] = {(word[i] & 0x000f000fu) | 0x64006400u, (word[i] & 0x00f000f0u) | 0x64006400u,
                           (up & 0x000f000fu) | 0x64006400u, (up & 0x00f000f0u) | 0x64006400u};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            __half2 x = *reinterpret_cast<__half2*>(&e[q]);
            x = (q & 1) ? __hfma2(x, R, B) : __hadd2(x, A);  // code - zero point, exactly
            x = __hmul2(x, S);
            e[q] = *reinterpret_cast<uint32_t*>(&x);
          }
          sts128(dst + to[i] + j * STEP * 128, e[0], e[1], e[2], e[3]);
        }
      }
      fence_proxy_async();
      mbar_arrive(&kv_full[s]);
    }
  } else {
    // ---- softmax: one warpgroup per tile, one row (TMEM lane) per thread -------------------------------
    const int t = (warp - 8) >> 2;
    const int q = warp & 3;  // TMEM lane quadrant this warp may touch
    const int rit = q * 32 + lane;
    const int tok = rit / p.hq, head = rit % p.hq;
    const float sc2 = p.scale * LOG2E;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t tmem_s = tmem + lane_base + t * 128;
    const uint32_t tmem_o = tmem + lane_base + 256 + t * D;
    int base = 0, unit = 0;
    do {
      const int nt = subs_of(p, w, t);
      const int local = w.i * 2 * p.tm + (w.narrow ? 0 : t * p.tm) + tok;  // the row within its piece
      const bool live = tok < p.tm && local < w.r.nrows;
      const int row = w.r.pos0 + local;
      float m_ref = -1e30f, l = 0.f;
      for (int n = 0; n < nt; ++n) {
        const int cnt = base + n, b = cnt & 1;
        const int key0 = w.k0 * CQ_BN + (w.narrow ? 2 * n + t : n) * CQ_SN;
        mbar_wait(&s_full[t * 2 + b], (cnt >> 1) & 1, p.status, 608);
        tc_fence_after();
        uint32_t sv[CQ_SN];
#pragma unroll
        for (int c = 0; c < CQ_SN / 32; ++c) tmem_ld32(tmem_s + b * CQ_SN + c * 32, sv + c * 32);
        tmem_ld_wait();
        float mx;
        if (key0 + CQ_SN - 1 <= row) {
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < CQ_SN; i += 4)
#pragma unroll
            for (int u = 0; u < 4; ++u) m4[u] = fmaxf(m4[u], __uint_as_float(sv[i + u]));
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        } else {
          mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < CQ_SN; ++i) {
            const float x = key0 + i <= row ? __uint_as_float(sv[i]) : -INFINITY;
            sv[i] = __float_as_uint(x);
            mx = fmaxf(mx, x);
          }
        }
        mx = fmaf(mx, sc2, -P_AIM);  // log2 domain (the scale is positive)
        const float m_new = fmaxf(m_ref, mx);
        const bool grow = m_new > m_ref + RESCALE_STEP;
        if (n == 0) {
          m_ref = m_new;
        } else if (__any_sync(0xffffffffu, grow)) {
          // O must be quiescent: S(n) was issued behind P V(n - 2), so only P V(n - 1) can still run.
          mbar_wait(&o_done[t * 2 + ((cnt - 1) & 1)], ((cnt - 1) >> 1) & 1, p.status, 609);
          tc_fence_after();
          const float f = grow ? exp2f(m_ref - m_new) : 1.0f;
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 8) {
            uint32_t ov[8];
            tmem_ld8(tmem_o + c0, ov);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
            tmem_st8(tmem_o + c0, ov);
          }
          l *= f;
          if (grow) m_ref = m_new;
        }
        uint64_t sum[2] = {0, 0};  // two pairs of partial sums
        const uint64_t by = pair2(sc2, sc2), less = pair2(-m_ref, -m_ref);
        // Eight columns at a time, so that scores and weights are not all live at once. (All scores are in
        // registers: overwriting the buffer's first columns loses nothing.)
#pragma unroll
        for (int c = 0; c < CQ_SN / 16; ++c) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a, b2;
            split2(fma2(pair2(__uint_as_float(sv[16 * c + 2 * i]), __uint_as_float(sv[16 * c + 2 * i + 1])), by, less), a, b2);
            a = ex2(a), b2 = ex2(b2);
            sum[i & 1] = add2(sum[i & 1], pair2(a, b2));
            pk[i] = pack_h2(a, b2);
          }
          tmem_st8(tmem_s + b * CQ_SN + 8 * c, pk);
        }
        float s0, s1;
        split2(add2(sum[0], sum[1]), s0, s1);
        tmem_st_wait();
        l += s0 + s1;
        tc_fence_before();
        mbar_arrive(&p_ready[t * 2 + b]);
      }
      if (nt > 0) {
        // The last two products may still be running.
        const int cnt = base + nt;
        if (nt > 1) mbar_wait(&o_done[t * 2 + ((cnt - 2) & 1)], ((cnt - 2) >> 1) & 1, p.status, 610);
        mbar_wait(&o_done[t * 2 + ((cnt - 1) & 1)], ((cnt - 1) >> 1) & 1, p.status, 611);
        tc_fence_after();
      }
      const bool whole = w.k0 == 0 && w.k1 == w.tiles;
      // A narrow unit's tiles agree on a maximum; the first takes the second's rows, which lie in the same
      // lanes of tensor memory, with its own.
      float mine = 1.0f, others = 0.f;
      if (w.narrow) {
        float* ex = (float*)(smem + SM::OFF_EX);
        ex[t * 128 + rit] = m_ref;
        if (t == 1) ex[256 + rit] = l;
        tc_fence_before();
        asm volatile("bar.sync 2, 256;" ::: "memory");
        tc_fence_after();
        if (t == 0) {
          const float mo = ex[128 + rit], m2 = fmaxf(m_ref, mo);
          mine = exp2f(m_ref - m2);
          if (subs_of(p, w, 1) > 0) others = exp2f(mo - m2), l = l * mine + ex[256 + rit] * others;
          m_ref = m2;
        }
      }
      const bool joins = others != 0.f || l != l;  // (a NaN sum comes with NaN rows)
      const bool stores = live && !(w.narrow && t == 1);
      const float inv = 1.0f / l;
      __half* o = p.O + ((size_t)(w.r.row0 + local) * p.H + w.g * p.hq + head) * D;
      // A partial: a column at a time, a warp's rows side by side: full lines.
      float* part = p.part + ((size_t)blockIdx.x * 2 + (w.k0 == 0 ? 1 : 0)) * 256 * (D + 2) + (w.narrow ? 0 : t * 128) + rit;
      const bool second = w.narrow && t == 0 && subs_of(p, w, 1) > 0;
#pragma unroll 1
      for (int c0 = 0; c0 < D && !(w.narrow && t == 1); c0 += 8) {
        uint32_t ov[8], ow[8];
        if (nt > 0) tmem_ld8(tmem_o + c0, ov);
        if (second) tmem_ld8(tmem_o + D + c0, ow);
        tmem_ld_wait();
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = nt > 0 ? __uint_as_float(ov[i]) * mine : 0.f;
          if (second && joins) y[i] = fmaf(__uint_as_float(ow[i]), others, y[i]);
        }
        if (stores) {
          if (nan_at[(unit & 7) * 2 + (c0 >> 6)] <= row) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7fc00000);
          }
          if (whole) {
            uint4 h;
            h.x = pack_h2(y[0] * inv, y[1] * inv), h.y = pack_h2(y[2] * inv, y[3] * inv);
            h.z = pack_h2(y[4] * inv, y[5] * inv), h.w = pack_h2(y[6] * inv, y[7] * inv);
            *reinterpret_cast<uint4*>(o + c0) = h;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) part[(size_t)(c0 + i) * 256] = y[i];
          }
        }
      }
      if (!whole) {
        if (stores) part[D * 256] = m_ref, part[(D + 1) * 256] = l;
        if (t == 0 && rit == 0 && w.k0 == 0) {
          // Cut at this CTA's end: the next CTAs go on with it.
          int* d = p.desc + 4 * blockIdx.x;
          d[0] = w.c, d[1] = w.g, d[2] = w.i;
          d[3] = 1 + (int)((w.tiles - w.k1 + w.share - 1) / w.share);
        }
      }
      base += nt;
      // This unit's marks are free again once all softmax threads are through with them. The unpacking
      // warps are at most three units (six tiles) ahead of the products: eight sets are enough.
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (threadIdx.x == 256) nan_at[(unit & 7) * 2] = nan_at[(unit & 7) * 2 + 1] = 0x7fffffff;
      ++unit;
    } while (w.next(p));
  }
  tc_fence_before();
  __syncthreads();
  pdl_launch();  // only now: a dependent's CTA let in earlier would wait for this one's shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, SM::TMEM_COLS);
  }
}

// Joins the partials of the unit that is cut at the end of CTA blockIdx.x, if there is one: that
// CTA's second slot and the first slots of the CTAs that follow. A thread joins eight columns of a row;
// the block's y says which.
template <int D>
__global__ void __launch_bounds__(256) chunk_q4_join_kernel(const CqParams p) {
  pdl_wait();
  pdl_launch();
  const int* d = p.desc + 4 * blockIdx.x;
  const int c = d[0], g = d[1], i = d[2], pieces = d[3];
  if (pieces < 2) return;
  const Piece r = piece_of(p, c);
  const int rr = threadIdx.x, t = rr >> 7, tok = (rr & 127) / p.hq, head = (rr & 127) % p.hq;
  const int local = i * 2 * p.tm + t * p.tm + tok;
  if (tok >= p.tm || local >= r.nrows) return;
  constexpr int U = 3;  // partials in flight
  float m = -1e30f, l = 0.f, a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = 0.f;
  for (int k0 = 0; k0 < pieces; k0 += U) {
    float v[U][8], mk[U], lk[U], m2 = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u;
      const bool in = k < pieces;
      const float* s = p.part + ((size_t)(blockIdx.x + (in ? k : 0)) * 2 + (k == 0 ? 1 : 0)) * 256 * (D + 2) + rr;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = in ? s[(size_t)(blockIdx.y * 8 + e) * 256] : 0.f;
      mk[u] = in ? s[D * 256] : -1e30f, lk[u] = in ? s[(D + 1) * 256] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) m2 = fmaxf(m2, mk[u]);
    const float f = ex2(m - m2);
    l *= f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float fk = ex2(mk[u] - m2);
      l = fmaf(lk[u], fk, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = fmaf(v[u][e], fk, a[e]);
    }
    m = m2;
  }
  uint4 y;
  y.x = pack_h2(a[0] / l, a[1] / l), y.y = pack_h2(a[2] / l, a[3] / l);
  y.z = pack_h2(a[4] / l, a[5] / l), y.w = pack_h2(a[6] / l, a[7] / l);
  *reinterpret_cast<uint4*>(p.O + ((size_t)(r.row0 + local) * p.H + g * p.hq + head) * D + blockIdx.y * 8) = y;
}

}  // namespace

bool chunk_q4_takes(const Q4Shape& q, int T, int H, int C, int MP) {
  return q.P == 16 && (q.D == 64 || q.D == 128) && q.NP > 0 && MP > 0 && T > 0 && C > 0 && H / q.G <= CQ_BM;
}

size_t chunk_q4_workspace(const Ctx* c, int D) { return (size_t)c->sm_count * (2 * 256 * (D + 2) * sizeof(float) + 16); }

int make_chunk_q4(Ctx* c, Op& op, const Q4Shape& q) {
  op.p1 = c->sm_count;
  if (q.D == 128)
    TB_CUDA(c, cudaFuncSetAttribute(chunk_q4_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, CqSmem<128>::TOTAL));
  else
    TB_CUDA(c, cudaFuncSetAttribute(chunk_q4_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, CqSmem<64>::TOTAL));
  return 0;
}

int launch_chunk_q4(Ctx* c, Op& op, const uint64_t* a, const Q4Shape& q) {
  const auto& s = op.shapes;
  CqParams p;
  p.T = (int)s[0][0], p.H = (int)s[0][1], p.G = q.G, p.hq = p.H / p.G, p.tm = CQ_BM / p.hq;
  p.C = (int)s[4][0], p.NP = q.NP, p.MP = (int)s[3][1];
  // Q [T, H, D]: one box = the group's heads of tm tokens, 64 columns.
  const uint64_t dims[3] = {(uint64_t)q.D, (uint64_t)p.H, (uint64_t)p.T};
  const uint64_t strides[2] = {(uint64_t)q.D * 2, (uint64_t)p.H * q.D * 2};
  const uint32_t box[3] = {64, (uint32_t)p.hq, (uint32_t)p.tm};
  CUtensorMap map;
  if (make_tensor_map(c, &map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (const void*)a[0], dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
    return 1;
  p.Kc = (const unsigned char*)a[1];
  p.Vc = (const unsigned char*)a[2];
  p.table = (const int*)a[3];
  p.meta = (const int*)a[4];
  p.O = (__half*)a[5];
  p.scale = bits_f32(a[6]);
  p.status = c->status;
  p.part = (float*)c->q4_work[q.D == 128];
  p.desc = (int*)(p.part + (size_t)op.p1 * 2 * 256 * (q.D + 2));
  const dim3 grid(op.p1), join(op.p1, q.D / 8);
  if (q.D == 128) {
    TB_CUDA(c, launch_k(c, chunk_q4_kernel<128>, grid, dim3(CQ_THREADS), CqSmem<128>::TOTAL, 1, map, p));
    TB_CUDA(c, launch_k(c, chunk_q4_join_kernel<128>, join, dim3(256), 0, 1, p));
  } else {
    TB_CUDA(c, launch_k(c, chunk_q4_kernel<64>, grid, dim3(CQ_THREADS), CqSmem<64>::TOTAL, 1, map, p));
    TB_CUDA(c, launch_k(c, chunk_q4_join_kernel<64>, join, dim3(256), 0, 1, p));
  }
  c->launches += 2;
  return 0;
}

}  // namespace tb
