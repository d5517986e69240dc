// Paged grouped-query decode attention over the 4-bit cache (format: kv_q4.cuh), for pages of 16
// tokens and head_dim 64 or 128; other shapes run on kv_q4.cu's one-warp kernel.
//
// Mathematics. With a key's code u, zero point z and scale s (64 elements share z and s), and a
// query q: q.k = sum over groups of s (q.u - z sum(q)); so the tensor cores multiply q by the raw
// codes and the scale and zero point come in afterwards, once per (token, head, group). For the
// values, o = sum_t p_t s_t (u_t - z_t) = sum_t P_t u_t - sum_t P_t z_t with P = p s: the scale rides on
// the weight, the second sum is one number per (head, group).
//
// The tensor cores cut products and sums off towards zero, and products that are never negative would
// grow hundreds of times larger than the result of a long context, all of them cut down. So the tokens
// of the second half of a page enter as (-P)(15 - u), with P (15 - z) in the other sum: the complement
// costs no instruction, products of both signs nearly cancel, and so do their cuts. What the other sum
// still holds is taken out of the accumulators every CENTRE pairs of pages. (Four of 131072 tokens, 32/8
// heads: 2.11e-4 off in all, of which 2.108e-4 by rounding to f16; 2.8e-4 without the complement.)
//
// A code becomes an f16 operand by one AND: the nibble in the low bits of an f16 is the subnormal
// u 2^-24, the next nibble 16 u 2^-24, and the tensor cores take subnormals as they are. For the
// keys the 16 is in q: 16 q meets the low nibbles, q the high ones, both exact. (Where a head group holds
// a |q| of 4096 or more, 16 q may pass the largest f16: there q and q / 16, which loses bits of numbers
// below 2^-22 of that one.) For the values it is taken out of the accumulators.
//
// P is split in two f16 (hi + lo): 22 bits down to 2^-2, below that the multiples of 2^-24. A power of
// two F for each head and group follows the largest P, up and down: not the largest scale, nor another
// head's or group's, for a token of great weight and no value, or a group of far larger values, must not
// push the other P off that grid. The largest P of a head and group is about 2^10 or more, so what the
// grid cuts off a weight is less than 2^-34 of it. All sums take the P that is left on the grid: a weight
// that falls off it is left out, where a sum of u without it and one of z with it would leave -z.
//
// The eight columns of a product. With four or fewer query heads per KV head (SIDE) q stands in them
// twice and a warp takes two pages at a time: columns 0..3 of the first page's scores and 4..7 of the
// second's go on, so no lane of the softmax does another's work; and the hi and lo parts of P share a
// product, side by side. With five to eight heads a page fills the columns,
// and lo is a second product.
//
// Bound: by bytes 2 (D/2 + 2 D/64) per token and KV head, from HBM. Measured, nothing is saturated (HBM 0.64 of the copy
// rate, integer pipe 58 %, issue slots 51 %): what is left is latency that fewer than three warps per scheduler
// do not hide. 256 sequences of 512-2304 tokens, 32/8 heads, D 128: 97 us as calls on changing inputs, 3.9 TB/s
// (93 with the same launches back to back); 4 of 100000-131072: 118 us, 4.2 TB/s (110). SM clock 1965 MHz.
//
// Work split. Every warp works on its own: it takes an equal share of the step's (sequence, KV head,
// page) list, whatever the lengths are, finds its place from the lengths, brings its pages through a
// ring of its own (bulk copies it issues itself, a few pairs of pages ahead, across units), and
// writes O for units that lie wholly inside its share. A unit that is cut leaves one partial with
// each warp; a second, tiny kernel joins them. Where the KV heads are even in number, two or four
// neighbouring warps take neighbouring heads of the same pages: their records lie side by side, and
// DRAM delivers neighbours that are asked for together faster than records picked one by one.
#include "kv_q4.cuh"

namespace tb {

namespace {

constexpr int DQ_WARPS = 4;
constexpr int DQ_THREADS = DQ_WARPS * 32;
static_assert(DQ_WARPS % 4 == 0, "sets of one, two or four head groups divide a CTA's warps");
constexpr int DQ_STAGES = 4;  // pairs of pages in a ring
constexpr int DQ_CTAS = 3;    // per SM
constexpr int DQ_LEAST = 2;   // pages a warp takes at least: a pair
constexpr int DQ_SLOT = 8;    // heads of a partial
constexpr float LOG2E = 1.4426950408889634f;
constexpr float TWO24 = 16777216.0f;
constexpr float NO_MAX = -1e30f;    // the running maximum before the first page
constexpr float GROW = 8.0f;        // the running maximum is renewed when a score passes it by this (log2): p <= 2^8
constexpr float P_MOST = 32768.f;   // and F when a P = p s F reaches this, to put the largest at 2^P_AIM or more
constexpr int P_AIM = 10;
constexpr int F_MOST = 100;         // log2 of the largest F, and the first: s F p < 2^(14 + 100 + 8) is finite

constexpr int CENTRE = 8;            // pairs of pages between two centrings of the accumulators

// What a table entry outside the cache reads as.
__device__ __align__(128) unsigned char g_zero_record[4608];

struct DqParams {
  const __half* Q;
  const unsigned char* Kc;
  const unsigned char* Vc;
  const int* table;
  const int* lens;
  __half* O;
  float* part;  // [warp][2][8][D + 2]: accumulators [8][D], then maxima [8] and sums [8]
  int* desc;    // [warp][4]: sequence, head group, warps that hold a piece of the unit cut at this warp's end (0: none)
  float scale;
  int B, H, G, NP, MP, hgroups;
  int units;  // sets of WH head groups, which neighbouring warps take side by side, in a sequence
  unsigned int* status;
};

template <int D>
struct DqSmem {
  static constexpr int REC = 16 * (D / 2 + 2 * (D / 64));
  static constexpr int PAGE = 2 * REC;  // K and V of a page
  static constexpr int STAGE = 2 * PAGE;
  static constexpr int RING = DQ_STAGES * STAGE;  // a warp's part of its set's ring
  static constexpr int BARS = DQ_WARPS * RING;
  static constexpr int SCAN = BARS + 2 * DQ_WARPS * DQ_STAGES * 8;  // long long [DQ_THREADS + 1], then the sets' places
  static constexpr int TOTAL = SCAN + (DQ_THREADS + 1 + 2 * DQ_WARPS) * 8 + 128;
};

__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float lo_f32(uint32_t h2) { return __low2float(*reinterpret_cast<__half2*>(&h2)); }
__device__ __forceinline__ float hi_f32(uint32_t h2) { return __high2float(*reinterpret_cast<__half2*>(&h2)); }

// A place in the list of (sequence, set of head groups, page): sequences in order, the sets of one
// after another, its pages within.
struct Place {
  int b, hg, page;
};

__device__ __forceinline__ long long pages_of(int n) { return n > 0 ? ((long long)n + 15) / 16 : 0; }

// The number of (unit, page) items, the share of a set of WH warps, and where this one begins. All
// threads call it.
template <int WH>
__device__ __forceinline__ Place find_place(const DqParams& p, long long* scan, long long* total, long long* share) {
  constexpr int owners = DQ_WARPS / WH;
  const int units = p.units, lane = threadIdx.x & 31;
  const int per = (p.B + DQ_THREADS - 1) / DQ_THREADS;
  const int b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) sum += pages_of(p.lens[b]);
  // Exclusive prefix of the threads' sums.
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scan[threadIdx.x >> 5] = inc;
  __syncthreads();
  long long before = inc - sum, pages = 0;
#pragma unroll
  for (int w = 0; w < DQ_WARPS; ++w) {
    if (w < (int)(threadIdx.x >> 5)) before += scan[w];
    pages += scan[w];
  }
  const long long all = pages * units, workers = (long long)gridDim.x * owners;
  const long long s = max((all + workers - 1) / workers, (long long)DQ_LEAST);
  *total = all;
  *share = s;
  // The thread whose sequences hold a warp's start says which one.
  long long at = before * units;
  for (int b = b0; b < b1; ++b) {
    const long long end = at + pages_of(p.lens[b]) * units;
#pragma unroll
    for (int w = 0; w < owners; ++w) {
      const long long start = ((long long)blockIdx.x * owners + w) * s;
      if (start >= at && start < end) {
        scan[DQ_WARPS + 2 * w] = b;
        scan[DQ_WARPS + 2 * w + 1] = start - at;
      }
    }
    at = end;
  }
  __syncthreads();
  Place r = {0, 0, 0};
  const int own = (threadIdx.x >> 5) / WH;
  if (((long long)blockIdx.x * owners + own) * s < all) {
    r.b = (int)scan[DQ_WARPS + 2 * own];
    const long long np = pages_of(p.lens[r.b]), in = scan[DQ_WARPS + 2 * own + 1];
    r.hg = (int)(in / np);
    r.page = (int)(in % np);
  }
  return r;
}

// A walk along a warp's share: the current unit's pages [at.page, at.page + count) are its own.
struct Walk {
  Place at;
  int left, np, n, count;
  __device__ __forceinline__ void set(const DqParams& p) {
    n = p.lens[at.b];
    while (n <= 0) n = p.lens[++at.b];  // (only at the start of a sequence; `left` says that one follows)
    np = (int)pages_of(n);
    count = min(np - at.page, left);
    left -= count;
  }
  // To the next unit; false at the end of the share.
  __device__ __forceinline__ bool next(const DqParams& p, int units) {
    if (left <= 0) return false;
    at.page = 0;
    if (++at.hg == units) at.hg = 0, ++at.b;
    set(p);
    return true;
  }
};

template <int D, bool SIDE, int WH>
__global__ void __launch_bounds__(DQ_THREADS, DQ_CTAS) decode_q4_kernel(const DqParams p) {
  using SM = DqSmem<D>;
  constexpr int NG = D / 64;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 127) & ~(uintptr_t)127);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int worker = blockIdx.x * DQ_WARPS + warp;
  const int own = warp / WH, wh = warp % WH;  // this warp's set, and its head group in it
  unsigned char* ring = smem + own * (WH * SM::RING);
  uint64_t* full = (uint64_t*)(smem + SM::BARS) + own * DQ_STAGES;
  uint64_t* empty = (uint64_t*)(smem + SM::BARS) + (DQ_WARPS + own) * DQ_STAGES;
  if (lane == 0) {
    if (wh == 0) {
      for (int s = 0; s < DQ_STAGES; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], WH);
      }
      fence_barrier_init();
    }
  }
  pdl_wait();
  if (lane == 0) p.desc[4 * worker + 2] = 0;
  long long total, share;
  Walk w;
  w.at = find_place<WH>(p, (long long*)(smem + SM::SCAN), &total, &share);
  const long long first = (long long)(worker / WH) * share;
  w.left = first < total ? (int)min(share, total - first) : 0;  // (2^31 pages for one warp would be hours of work)
  const int units = p.units, hq = p.H / p.G;
  bool busy = w.left > 0;
  if (busy) w.set(p);

  // ---- loads: `lw` walks the same units ahead of `w`. The set's warps take turns: one of them brings a
  // pair of pages for all, the records of the set's KV heads in one copy per page and cache. ------------
  Walk lw = w;
  bool more = busy;
  int lpair = 0, ls = 0, lphase = 1, turn = 0;  // the pair of its unit that comes next, its slot, and whose turn it is
  int tab = 0, tab_next = 0;                    // the block table's entries of 16 pairs, a page per lane, and of the next 16
  const int rec_page = p.G * SM::REC;
  size_t aim = 0;   // the set's first KV head within a page
  int heads_b = 0;  // and the bytes of its KV heads (head groups of one KV head share them)
  auto take_aim = [&]() {
    const int k0 = lw.at.hg * WH / p.hgroups, k1 = (lw.at.hg * WH + WH - 1) / p.hgroups;
    aim = (size_t)k0 * SM::REC;
    heads_b = (k1 - k0 + 1) * SM::REC;
  };
  auto entries = [&](int pair) {
    const int i = 2 * pair + lane, col = lw.at.page + i;  // beyond the table: page 0
    return i < lw.count && col < p.MP ? p.table[(size_t)lw.at.b * p.MP + col] : 0;
  };
  auto load = [&]() {
    if (!more) return;
    if ((lpair & 15) == 0) {
      tab = lpair == 0 ? entries(0) : tab_next;
      if (2 * (lpair + 16) < lw.count) tab_next = entries(lpair + 16);
    }
    const int pages = min(2, lw.count - 2 * lpair);
    if (WH == 1 || turn == wh) {
      const int pa = __shfl_sync(0xffffffffu, tab, 2 * (lpair & 15)), pb = __shfl_sync(0xffffffffu, tab, 2 * (lpair & 15) + 1);
      if (elect_one()) {
        unsigned char* dst = ring + ls * (WH * SM::STAGE);
        mbar_wait(&empty[ls], lphase, p.status, 501);
        mbar_expect_tx(&full[ls], pages * 2 * heads_b);
        const bool in_a = (unsigned)pa < (unsigned)p.NP, in_b = (unsigned)pb < (unsigned)p.NP;
        const size_t off_a = aim + (long long)pa * rec_page, off_b = aim + (long long)pb * rec_page;
        bulk_load(dst, in_a ? p.Kc + off_a : g_zero_record, heads_b, &full[ls]);
        bulk_load(dst + WH * SM::REC, in_a ? p.Vc + off_a : g_zero_record, heads_b, &full[ls]);
        if (pages == 2) {
          bulk_load(dst + WH * SM::PAGE, in_b ? p.Kc + off_b : g_zero_record, heads_b, &full[ls]);
          bulk_load(dst + WH * (SM::PAGE + SM::REC), in_b ? p.Vc + off_b : g_zero_record, heads_b, &full[ls]);
        }
      }
      __syncwarp();
    }
    if (WH > 1) turn = (turn + 1) % WH;
    if (++ls == DQ_STAGES) ls = 0, lphase ^= 1;
    if (2 * ++lpair >= lw.count) {
      lpair = 0;
      more = lw.next(p, units);
      take_aim();
    }
  };
  take_aim();
  // Two pairs ahead: the slot that is filled next was read a pair ago, so that the set's warps need not
  // keep pace exactly.
  for (int i = 0; i < DQ_STAGES - 2; ++i) load();

  const int gq = lane >> 2, t = lane & 3;
  // Rows of the K tile (and columns of the V tile) are the page's tokens in the order that lets a
  // lane's four V tokens be t, 4 + t, 8 + t, 12 + t: row r is token (r & 7) / 2 + 4 (r & 1) + (r & 8).
  const int tok_a = (gq >> 1) + 4 * (gq & 1), tok_b = tok_a + 8;
  const uint32_t ring_u = smem_u32(ring);
  const int side = SIDE ? t >> 1 : 0;  // the page of a pair whose scores this lane holds
  int cs = 0, phase = 0;               // the slot that is read next, and its phase
  for (; busy; busy = w.next(p, units)) {
    const Place& at = w.at;
    const int n = w.n, count = w.count, pairs = (count + 1) / 2;
    // Tokens of this segment: those behind it are another CTA's, or do not exist.
    const int tokens = (int)min(16LL * count, n - 16LL * at.page);
    const int hg = at.hg * WH + wh;
    const uint32_t mine = (hg / p.hgroups - at.hg * WH / p.hgroups) * SM::REC;  // this head's record in a slot
    const int h0 = hg / p.hgroups * hq + (hg % p.hgroups) * 8, nh = min(8, hq - (hg % p.hgroups) * 8);

    // Q as the B operand: column gq is head gq (SIDE: head gq & 3), the rows of step k of group x are elements
    // 64 x + 16 t + 2 k, + 1 and the same + 8, as the words of codes hold them; odd steps' nibbles weigh 16.
    uint32_t qf[NG][4][2];
    float qsum[NG][2], sc2 = p.scale * LOG2E * TWO24;
    {
      bool large = false;  // some |q| is 4096 or more
      const int hc = SIDE ? gq & 3 : gq;
      const bool live = hc < nh;
      const __half* q = p.Q + ((size_t)at.b * p.H + h0 + (live ? hc : 0)) * D + 16 * t;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (live) {
          lo = *reinterpret_cast<const uint4*>(q + 64 * x);
          hi = *reinterpret_cast<const uint4*>(q + 64 * x + 8);
        }
        const uint32_t w[4][2] = {{lo.x, hi.x}, {lo.y, hi.y}, {lo.z, hi.z}, {lo.w, hi.w}};
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          s += lo_f32(w[k][0]) + hi_f32(w[k][0]) + lo_f32(w[k][1]) + hi_f32(w[k][1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            qf[x][k][e] = w[k][e];
            large = large || (w[k][e] & 0x7fffu) >= 0x6c00u || (w[k][e] & 0x7fff0000u) >= 0x6c000000u;
          }
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        qsum[x][0] = __shfl_sync(0xffffffffu, s, 8 * t);      // of column 2t
        qsum[x][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);  // of column 2t + 1
      }
      large = __any_sync(0xffffffffu, large);
      const uint32_t by = large ? 0x2c002c00u : 0x4c004c00u;  // 1 / 16, 16
#pragma unroll
      for (int x = 0; x < NG; ++x) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (((k & 1) != 0) == large) qf[x][k][e] = mul_h2(qf[x][k][e], by);
        if (!large) qsum[x][0] *= 16.f, qsum[x][1] *= 16.f;
      }
      if (!large) sc2 *= 0.0625f;
    }
    float m[2] = {NO_MAX, NO_MAX}, l[2] = {0.f, 0.f};
    float F[NG][2];  // of the columns' heads: the first page with a value sets it
    float acc[4 * NG][4], zsum[NG][2];  // zsum: P z, or P (z - 15), since the last centring, of this lane's tokens
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      zsum[x][0] = zsum[x][1] = 0.f;
      F[x][0] = F[x][1] = __uint_as_float((127u + F_MOST) << 23);
    }

    // One product's worth of tokens: a page, or (SIDE) a pair of pages at `pg`, `limit` tokens of them.
    auto tile = [&](uint32_t pg, int limit) {
      const uint32_t page = pg + side * (WH * SM::PAGE);  // the page of this lane's scores
      uint32_t hka, hkb, hva, hvb;  // headers of its two tokens: a pair of f16 (or one)
      if (NG == 2) {
        hka = lds32(page + 8 * D + 4 * tok_a), hkb = lds32(page + 8 * D + 4 * tok_b);
        hva = lds32(page + WH * SM::REC + 8 * D + 4 * tok_a), hvb = lds32(page + WH * SM::REC + 8 * D + 4 * tok_b);
      } else {
        hka = lds16(page + 8 * D + 2 * tok_a), hkb = lds16(page + 8 * D + 2 * tok_b);
        hva = lds16(page + WH * SM::REC + 8 * D + 2 * tok_a), hvb = lds16(page + WH * SM::REC + 8 * D + 2 * tok_b);
      }
      // Tokens behind the last one: stale headers may be NaN, and the scores are masked below.
      const bool tail = limit < (SIDE ? 32 : 16);
      const bool ok_a = 16 * side + tok_a < limit, ok_b = 16 * side + tok_b < limit;
      if (tail) {
        if (!ok_a) hka = hva = 0;
        if (!ok_b) hkb = hvb = 0;
      }
      constexpr int NS = SIDE ? 2 : 1;
      float e[NG][4];
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        float ep[NS][4];
        uint2 ua[NS], ub[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const uint32_t k0 = pg + s * (WH * SM::PAGE) + 32 * x + 8 * t;
          ua[s] = lds64(k0 + tok_a * (D / 2)), ub[s] = lds64(k0 + tok_b * (D / 2));
          ep[s][0] = ep[s][1] = ep[s][2] = ep[s][3] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            const uint32_t mask = (k & 1) ? 0x00f000f0u : 0x000f000fu;
            const int sh = 8 * (k >> 1);
            mma16816(ep[s], (ua[s].x >> sh) & mask, (ub[s].x >> sh) & mask, (ua[s].y >> sh) & mask, (ub[s].y >> sh) & mask,
                     qf[x][k][0], qf[x][k][1]);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) e[x][i] = SIDE && side ? ep[NS - 1][i] : ep[0][i];
      }
      // Scores of columns 2t, 2t + 1 in the log2 domain, less `from`.
      float xa[2], xb[2];
      auto scores = [&](float from0, float from1) {
        xa[0] = xb[0] = -from0, xa[1] = xb[1] = -from1;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const uint32_t sa = hka & 0xfff0fff0u, za = hka & 0x000f000fu, sb = hkb & 0xfff0fff0u, zb = hkb & 0x000f000fu;
          const float ka = (x ? hi_f32(sa) : lo_f32(sa)) * sc2, kza = x ? hi_f32(za) : lo_f32(za);
          const float kb = (x ? hi_f32(sb) : lo_f32(sb)) * sc2, kzb = x ? hi_f32(zb) : lo_f32(zb);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            xa[c] = fmaf(ka, fmaf(-kza, qsum[x][c], e[x][c]), xa[c]);
            xb[c] = fmaf(kb, fmaf(-kzb, qsum[x][c], e[x][2 + c]), xb[c]);
          }
        }
        if (tail) {
          if (!ok_a) xa[0] = xa[1] = -INFINITY;
          if (!ok_b) xb[0] = xb[1] = -INFINITY;
        }
      };
      scores(m[0], m[1]);
      // The running maximum is lazy: renewed (and the sums rescaled) only when a score outgrew it by 2^8.
      if (__any_sync(0xffffffffu, fmaxf(fmaxf(xa[0], xb[0]), fmaxf(xa[1], xb[1])) > GROW)) {
        scores(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(xa[c], xb[c]);
#pragma unroll
          for (int d = SIDE ? 2 : 4; d <= 16; d = d == 2 ? 4 : d * 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          mx = fmaxf(m[c], mx);
          const float by = m[c] - mx;
          m[c] = mx;
          l[c] *= ex2(by);
          // The sums lose a factor 2^by; F takes its whole powers of two, as far as it may.
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            const int up = min((int)fminf(rintf(-by), 300.f), 127 + F_MOST - (int)(__float_as_uint(F[x][c]) >> 23));
            const float f = ex2(by + (float)up);
            F[x][c] = __uint_as_float(__float_as_uint(F[x][c]) + ((uint32_t)up << 23));
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[4 * x + i][c] *= f, acc[4 * x + i][2 + c] *= f;
            zsum[x][c] *= f;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) xa[c] -= m[c], xb[c] -= m[c];  // (0 for the largest: a single token's weight is 1, its result its value)
      }
      const float pa[2] = {ex2(xa[0]), ex2(xa[1])}, pb[2] = {ex2(xb[0]), ex2(xb[1])};
      l[0] += pa[0] + pb[0];
      l[1] += pa[1] + pb[1];
      // P = p s F of the first token and -P of the second, columns in pairs.
      uint64_t wa[NG], wb[NG];
      {
        const uint32_t sa = hva & 0xfff0fff0u, sb = (hvb & 0xfff0fff0u) | 0x80008000u;
        const uint64_t p2a = pair2(pa[0], pa[1]), p2b = pair2(pb[0], pb[1]);
        float most = 0.f;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const float va = x ? hi_f32(sa) : lo_f32(sa), vb = x ? hi_f32(sb) : lo_f32(sb);
          const uint64_t f2 = pair2(F[x][0], F[x][1]);
          wa[x] = mul2(p2a, mul2(pair2(va, va), f2)), wb[x] = mul2(p2b, mul2(pair2(vb, vb), f2));
          float a0, a1, b0, b1;
          split2(wa[x], a0, a1);
          split2(wb[x], b0, b1);
          most = fmaxf(most, fmaxf(fmaxf(a0, a1), fmaxf(-b0, -b1)));
        }
        if (__any_sync(0xffffffffu, most >= P_MOST)) {
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            float a[2], b[2];
            split2(wa[x], a[0], a[1]);
            split2(wb[x], b[0], b[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mo = fmaxf(a[c], -b[c]);
#pragma unroll
              for (int d = SIDE ? 2 : 4; d <= 16; d = d == 2 ? 4 : d * 2) mo = fmaxf(mo, __shfl_xor_sync(0xffffffffu, mo, d));
              const uint32_t down = mo >= P_MOST ? (__float_as_uint(mo) >> 23) - 127u - P_AIM : 0u;
              const float f = __uint_as_float((127u - down) << 23);
              F[x][c] *= f, a[c] *= f, b[c] *= f;
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[4 * x + i][c] *= f, acc[4 * x + i][2 + c] *= f;
              zsum[x][c] *= f;
            }
            wa[x] = pair2(a[0], a[1]), wb[x] = pair2(b[0], b[1]);
          }
        }
      }
      uint32_t bf[NG][2][2];  // P as the B operand: SIDE: of either page; else its hi and its lo
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const uint32_t za = hva & 0x000f000fu, zb = hvb & 0x000f000fu;
        // z, and 15 - z where P is negative, 2^-24 each as the codes are.
        const float ca = x ? hi_f32(za) : lo_f32(za), cb = 15.f / TWO24 - (x ? hi_f32(zb) : lo_f32(zb));
        // To the grid: next to 0.75 a number below 0.25 keeps multiples of 2^-24 (a larger one its f32 bits, or 2^-23).
        const uint64_t grid = pair2(0.75f, 0.75f), off = pair2(-0.75f, -0.75f);
        float a0, a1, b0, b1;
        split2(add2(add2(wa[x], grid), off), a0, a1);
        split2(add2(add2(wb[x], off), grid), b0, b1);
        zsum[x][0] = fmaf(b0, cb, fmaf(a0, ca, zsum[x][0]));
        zsum[x][1] = fmaf(b1, cb, fmaf(a1, ca, zsum[x][1]));
        const uint32_t pha = pack_h2(a0, a1), phb = pack_h2(b0, b1);
        const uint32_t bh0 = movm_t(pha), bh1 = movm_t(phb);
        const uint32_t bl0 = movm_t(pack_h2(a0 - lo_f32(pha), a1 - hi_f32(pha)));
        const uint32_t bl1 = movm_t(pack_h2(b0 - lo_f32(phb), b1 - hi_f32(phb)));
        if (SIDE) {
          // Columns 0..3 of (bh, bl) are the first page's, 4..7 the second's. The first page's product takes
          // its hi in columns 0..3 and its lo in 4..7, the second's the other way round.
          const uint32_t ol0 = __shfl_xor_sync(0xffffffffu, bl0, 16), ol1 = __shfl_xor_sync(0xffffffffu, bl1, 16);
          bf[x][0][0] = gq < 4 ? bh0 : ol0, bf[x][0][1] = gq < 4 ? bh1 : ol1;
          bf[x][1][0] = gq < 4 ? ol0 : bh0, bf[x][1][1] = gq < 4 ? ol1 : bh1;
        } else {
          bf[x][0][0] = bh0, bf[x][0][1] = bh1, bf[x][1][0] = bl0, bf[x][1][1] = bl1;
        }
      }
#pragma unroll
      for (int x = 0; x < NG; ++x) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          // V^T: a lane's word gq of the group, for its four tokens; two tokens' halves side by side.
          const uint32_t v = pg + s * (WH * SM::PAGE) + WH * SM::REC + 32 * x + 4 * gq + t * (D / 2);
          const uint32_t w0 = lds32(v), w1 = lds32(v + 2 * D), w2 = lds32(v + 4 * D), w3 = lds32(v + 6 * D);
          const uint32_t lo01 = __byte_perm(w0, w1, 0x5410), hi01 = __byte_perm(w0, w1, 0x7632);
          const uint32_t lo23 = __byte_perm(w2, w3, 0x5410), hi23 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // Of the word's nibbles e0 e2 e4 e6 e1 e3 e5 e7: k = 0: e0, e2 are rows gq, gq + 8; 1: e4, e6; 2: e1,
            // e3; 3: e5, e7. Rows 8..15 always weigh 16.
            const uint32_t v01 = (k & 2 ? hi01 : lo01) >> (8 * (k & 1)), v23 = (k & 2 ? hi23 : lo23) >> (8 * (k & 1));
            const uint32_t a_0 = v01 & 0x000f000fu, a_1 = v01 & 0x00f000f0u, a_2 = ~v23 & 0x000f000fu, a_3 = ~v23 & 0x00f000f0u;
            mma16816(acc[4 * x + k], a_0, a_1, a_2, a_3, bf[x][s][0], bf[x][s][1]);
            if (!SIDE) mma16816(acc[4 * x + k], a_0, a_1, a_2, a_3, bf[x][1][0], bf[x][1][1]);
          }
        }
      }
    };

    auto centre = [&]() {
#pragma unroll
      for (int x = 0; x < NG; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float z = zsum[x][c];
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
          zsum[x][c] = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            acc[4 * x + k][c] -= z;
            acc[4 * x + k][2 + c] = fmaf(z, -16.f, acc[4 * x + k][2 + c]);
          }
        }
    };

    for (int j = 0; j < pairs; ++j) {
      load();
      const int limit = tokens - 32 * j;
      mbar_wait(&full[cs], phase, p.status, 502);
      const uint32_t pg = ring_u + cs * (WH * SM::STAGE) + mine;
      tile(pg, min(limit, 32));
      if (!SIDE && limit > 16) tile(pg + WH * SM::PAGE, min(limit - 16, 16));
      if ((j & (CENTRE - 1)) == CENTRE - 1 || j + 1 == pairs) centre();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[cs]);
      if (++cs == DQ_STAGES) cs = 0, phase ^= 1;
    }

    // ---- the segment's result ---------------------------------------------------------------------------
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = SIDE ? 2 : 4; d <= 16; d = d == 2 ? 4 : d * 2) l[c] += __shfl_xor_sync(0xffffffffu, l[c], d);
    const bool whole = at.page == 0 && count == w.np;
    float* part = p.part + ((size_t)worker * 2 + (at.page == 0 ? 1 : 0)) * DQ_SLOT * (D + 2);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int hh = (SIDE ? 2 * (t & 1) : 2 * t) + c;  // the head of this column
      const float inv = 1.0f / l[c];
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const float unit = TWO24 / F[x][c];
        float v[8];  // elements 64 x + 8 gq ...
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int upper = (i >> 1) & 1;  // the nibble's weight; its product: see above
          float a = acc[4 * x + 2 * (i & 1) + (i >> 2)][2 * upper + c];
          if (SIDE) a += __shfl_xor_sync(0xffffffffu, a, 2);  // columns h and h + 4 are the same head
          v[i] = a * (upper ? 0.0625f * unit : unit);
        }
        // SIDE: both lanes of a pair hold the sums; they take a group each.
        if (hh < nh && (!SIDE || (t >> 1) == x)) {
          const int d = 64 * x + 8 * gq;
          if (whole) {
            uint4 y;
            y.x = pack_h2(v[0] * inv, v[1] * inv), y.y = pack_h2(v[2] * inv, v[3] * inv);
            y.z = pack_h2(v[4] * inv, v[5] * inv), y.w = pack_h2(v[6] * inv, v[7] * inv);
            *reinterpret_cast<uint4*>(p.O + ((size_t)at.b * p.H + h0 + hh) * D + d) = y;
          } else {
            *reinterpret_cast<float4*>(part + hh * D + d) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(part + hh * D + d + 4) = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      if (!whole && gq == 0 && hh < nh && (!SIDE || t < 2)) part[DQ_SLOT * D + hh] = m[c], part[DQ_SLOT * (D + 1) + hh] = l[c];
    }
    if (lane == 0 && !whole && at.page == 0) {
      // The unit is cut at this warp's end: the next ones go on with it.
      int* d = p.desc + 4 * worker;
      d[0] = at.b, d[1] = hg;
      d[2] = 1 + (int)((w.np - count + share - 1) / share);
    }
  }

  // Only now: the next kernel's CTAs, let in earlier, would take the places of this one's and make the
  // equal shares unequal (256 sequences back to back: 229 us per launch instead of 149).
  pdl_launch();
  // Rows without a cached token: 0/0, as decode_attention gives.
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (p.lens[b] <= 0)
      for (int i = threadIdx.x; i < p.H * D; i += DQ_THREADS)
        p.O[(size_t)b * p.H * D + i] = __float2half_rn(__int_as_float(0x7fc00000));
}

// Joins the partials of the unit that is cut at the end of a warp's share, if there is one: that
// warp's second slot and the first slots of the warps that follow (`wh` apart). One block per share:
// HP heads, 8 / HP warps each, U partials in flight per warp (a long context has dozens).
template <int D, int HP>
__global__ void __launch_bounds__(256) decode_q4_join_kernel(const DqParams p, int wh) {
  pdl_wait();
  pdl_launch();
  constexpr int NSP = 8 / HP, V = D / 32, U = 4;
  __shared__ float other[8][D + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hh = warp % HP, sp = warp / HP;
  const int* d = p.desc + 4 * blockIdx.x;
  const int b = d[0], hg = d[1], pieces = d[2];
  if (pieces < 2) return;
  const int hq = p.H / p.G, h0 = (hg / p.hgroups) * hq + (hg % p.hgroups) * 8, nh = min(8, hq - (hg % p.hgroups) * 8);
  float m = NO_MAX, l = 0.f, a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  for (int i0 = sp; i0 < pieces && hh < nh; i0 += U * NSP) {
    float mi[U], li[U], ai[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NSP;
      const bool in = i < pieces;
      const float* s = p.part + ((size_t)(blockIdx.x + (in ? i : 0) * wh) * 2 + (in && i > 0 ? 0 : 1)) * DQ_SLOT * (D + 2);
      mi[u] = in ? s[DQ_SLOT * D + hh] : NO_MAX;
      li[u] = in ? s[DQ_SLOT * (D + 1) + hh] : 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) ai[u][k] = in ? s[hh * D + lane + 32 * k] : 0.f;
    }
    float m2 = m;
#pragma unroll
    for (int u = 0; u < U; ++u) m2 = fmaxf(m2, mi[u]);
    const float f = ex2(m - m2);
    l *= f;
#pragma unroll
    for (int k = 0; k < V; ++k) a[k] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float fu = ex2(mi[u] - m2);
      l = fmaf(li[u], fu, l);
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = fmaf(ai[u][k], fu, a[k]);
    }
    m = m2;
  }
  if (NSP > 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) other[warp][lane + 32 * k] = a[k];
    if (lane == 0) other[warp][D] = m, other[warp][D + 1] = l;
    __syncthreads();
    if (sp > 0) return;
#pragma unroll
    for (int o = 1; o < NSP; ++o) {
      const float* s = other[warp + o * HP];
      const float m2 = fmaxf(m, s[D]), f = ex2(m - m2), fo = ex2(s[D] - m2);
      l = fmaf(l, f, s[D + 1] * fo);
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = fmaf(a[k], f, s[lane + 32 * k] * fo);
      m = m2;
    }
  }
  if (hh >= nh) return;
#pragma unroll
  for (int k = 0; k < V; ++k)
    p.O[((size_t)b * p.H + h0 + hh) * D + lane + 32 * k] = __float2half_rn(a[k] / l);
}

int set_of(int sets) { return sets % 4 == 0 ? 4 : sets % 2 == 0 ? 2 : 1; }

// The kernel for a head_dim, at most four heads per KV head or more, and sets of one, two or four.
typedef void (*DqKernel)(DqParams);
template <int D>
DqKernel kernel_of(bool side, int wh) {
  if (side) return wh == 4 ? decode_q4_kernel<D, true, 4> : wh == 2 ? decode_q4_kernel<D, true, 2> : decode_q4_kernel<D, true, 1>;
  return wh == 4 ? decode_q4_kernel<D, false, 4> : wh == 2 ? decode_q4_kernel<D, false, 2> : decode_q4_kernel<D, false, 1>;
}
DqKernel kernel_of(int D, int hq, int wh) { return D == 128 ? kernel_of<128>(hq <= 4, wh) : kernel_of<64>(hq <= 4, wh); }

}  // namespace

bool decode_q4_takes(const Q4Shape& q, int B, int MP) {
  return q.P == 16 && (q.D == 64 || q.D == 128) && q.NP > 0 && B > 0 && MP > 0;
}

size_t decode_q4_workspace(const Ctx* c, int D) {
  return (size_t)c->sm_count * DQ_CTAS * DQ_WARPS * (2 * DQ_SLOT * (D + 2) * sizeof(float) + 16);
}

int make_decode_q4(Ctx* c, Op& op, const Q4Shape& q) {
  const int B = (int)op.shapes[0][0], H = (int)op.shapes[0][1];
  const int units = q.G * ((H / q.G + 7) / 8);
  // As many CTAs as stay resident, and no more than have DQ_LEAST pages to work on. (Lengths beyond
  // the table only make the shares larger.)
  const long long most = ((long long)B * units * op.shapes[3][1] + DQ_LEAST * DQ_WARPS - 1) / (DQ_LEAST * DQ_WARPS);
  const long long fit = (long long)c->sm_count * DQ_CTAS;
  op.p1 = (int)(most < fit ? most : fit);
  TB_CUDA(c, cudaFuncSetAttribute(kernel_of(q.D, H / q.G, set_of(units)), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  q.D == 128 ? DqSmem<128>::TOTAL : DqSmem<64>::TOTAL));
  return 0;
}

int launch_decode_q4(Ctx* c, Op& op, const uint64_t* a, const Q4Shape& q) {
  DqParams p;
  p.Q = (const __half*)a[0];
  p.Kc = (const unsigned char*)a[1];
  p.Vc = (const unsigned char*)a[2];
  p.table = (const int*)a[3];
  p.lens = (const int*)a[4];
  p.O = (__half*)a[5];
  p.scale = bits_f32(a[6]);
  p.B = (int)op.shapes[0][0], p.H = (int)op.shapes[0][1], p.G = q.G, p.NP = q.NP, p.MP = (int)op.shapes[3][1];
  p.hgroups = (p.H / p.G + 7) / 8;
  const int wh = set_of(p.G * p.hgroups);
  p.units = p.G * p.hgroups / wh;
  p.status = c->status;
  p.part = (float*)c->q4_work[q.D == 128];
  p.desc = (int*)(p.part + (size_t)op.p1 * DQ_WARPS * 2 * DQ_SLOT * (q.D + 2));
  const bool few = p.H / p.G <= 4;
  TB_CUDA(c, launch_k(c, kernel_of(q.D, p.H / p.G, wh), dim3(op.p1), dim3(DQ_THREADS),
                      q.D == 128 ? DqSmem<128>::TOTAL : DqSmem<64>::TOTAL, 1, p));
  TB_CUDA(c, launch_k(c, q.D == 128 ? (few ? decode_q4_join_kernel<128, 4> : decode_q4_join_kernel<128, 8>)
                                    : (few ? decode_q4_join_kernel<64, 4> : decode_q4_join_kernel<64, 8>),
                      dim3(op.p1 * DQ_WARPS), dim3(256), 0, 1, p, wh));
  c->launches += 2;
  return 0;
}

}  // namespace tb
