// The 4-bit KV cache: rope_q and the cache write of a step's rows (rope_kv_q4), rows read back as
// f16 (kv_unpack_q4), attention over it for every shape (the tensor-core kernels of
// decode_attention_q4.cu and chunk_attention_q4.cu take the common ones), and page_copy, which
// moves pages of any cache. The format is described in kv_q4.cuh.
#include "kv_q4.cuh"

namespace tb {

namespace {

// One step's QKV rows: Q rotated; K rotated, V as it is, both stored densely and, quantised, into
// their cache slots. The rotation rounds after every operation, as rope_kv does, so Q, K and V are
// that kernel's bit for bit.
//
// HBM-bound (at decode sizes: launch latency): the QKV row is read and the Q, K, V rows are written
// once, plus 4.25 bits per cached element. A row's work is a list of items: first the groups of its KV
// heads, eight lanes to a group's 64 elements (the bounds are three shuffles, a lane's codes one 32-bit
// store; the rotation partner lies D/2 away in the same row, both lanes load both halves), then the
// pairs of its query heads, eight to a thread. A thread keeps its place in the row and goes from row to
// row, so an item is taken apart once (64-bit divisions per item took a third of the time). x / scale
// is x times the reciprocal, corrected once by its exact remainder (Markstein): the quotient a division
// would give, for three instructions. 4352 rows of 32/8 heads, D 128: 24 us, 4.7 TB/s; what is left is a
// chain of latencies per row (position, rotation table, shuffles, slot) on 32 warps per SM.

// Both halves of a word as f32.
__device__ __forceinline__ uint64_t floats(uint32_t h2) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  return pair2(f.x, f.y);
}
// a b + c d as halves, each operation rounded by itself, as rope_kv does. (The additions stand alone: one of pairs
// behind two products of pairs was merged into an fma.)
__device__ __forceinline__ uint32_t rotated(uint64_t a, uint64_t b, uint64_t c, uint64_t d) {
  float x0, x1, y0, y1;
  split2(mul2(a, b), x0, x1);
  split2(mul2(c, d), y0, y1);
  return pack_h2(__fadd_rn(x0, y0), __fadd_rn(x1, y1));
}
// The larger of each half; NaN if either is.
__device__ __forceinline__ uint32_t max_h2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Eight numbers of a group as codes and (in lane 0 of eight) the group's header.
__device__ __forceinline__ void quantise8(const uint4& x, uint32_t& word, uint32_t& head) {
  const uint32_t h[4] = {x.x, x.y, x.z, x.w}, minus = 0x80008000u;
  // The largest of the numbers (low half) and of their negatives, and zero.
  const uint32_t up = max_h2(max_h2(h[0], h[1]), max_h2(h[2], h[3]));
  const uint32_t down = max_h2(max_h2(h[0] ^ minus, h[1] ^ minus), max_h2(h[2] ^ minus, h[3] ^ minus));
  uint32_t m = max_h2(0u, max_h2(__byte_perm(up, down, 0x5410), __byte_perm(up, down, 0x7632)));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max_h2(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool odd = (m & 0x7c00u) == 0x7c00u || (m & 0x7c000000u) == 0x7c000000u;  // an infinity or a NaN
  const float2 bound = __half22float2(*reinterpret_cast<const __half2*>(&m));
  head = odd ? 0x7e00u : q4_scale_bits(bound.x, bound.y);
  const float scale = q4_scale(head);
  word = 0;
  if (odd || scale == 0.f) return;
  const float r = __frcp_rn(scale);
  const uint64_t r2 = pair2(r, r), s2 = pair2(-scale, -scale);
  auto over = [&](uint64_t v) {
    const uint64_t q = mul2(v, r2);
    return fma2(fma2(q, s2, v), r2, q);
  };
  float zp, most;
  split2(over(pair2(bound.y, 65504.f)), zp, most);
  zp = fminf(rintf(zp), 15.f), most = floorf(most);
  // rint(x / scale) kept to +-most and its sum with zp to 0..15: the bounds are integers, so they may
  // come before the rounding. Adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the
  // low bits; the sum of eight such words, shifted to the codes' places, needs the zero points added and
  // the constants taken off only once, modulo 2^32.
  const float least = fmaxf(-most, -zp), largest = fminf(most, 15.f - zp);
  const uint64_t magic = pair2(12582912.0f, 12582912.0f);
  const uint32_t z = (uint32_t)zp;
  word = (z - 0x4b400000u) * 0x11111111u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    split2(over(floats(h[j])), a, b);
    split2(add2(pair2(fminf(fmaxf(a, least), largest), fminf(fmaxf(b, least), largest)), magic), a, b);
    word += (__float_as_uint(a) << (4 * j)) + (__float_as_uint(b) << (4 * j + 16));
  }
  head |= z;
}

// Eight elements of a rotation table as pairs; zeros for a position outside it.
__device__ __forceinline__ void load8(const float* __restrict__ p, bool in, uint64_t* o) {
  const ulonglong2 z = make_ulonglong2(0, 0), a = in ? *reinterpret_cast<const ulonglong2*>(p) : z,
                   b = in ? *reinterpret_cast<const ulonglong2*>(p + 4) : z;
  o[0] = a.x, o[1] = a.y, o[2] = b.x, o[3] = b.y;
}

constexpr int WRITE_THREADS = 128;

__global__ void __launch_bounds__(WRITE_THREADS)
    rope_kv_q4_kernel(const __half* __restrict__ QKV, const int* __restrict__ pos, const int* __restrict__ slot,
                      const float* __restrict__ Ct, const float* __restrict__ St, __half* __restrict__ Q,
                      unsigned char* __restrict__ Kc, unsigned char* __restrict__ Vc, __half* __restrict__ Kd,
                      __half* __restrict__ Vd, int T, int H, int NPOS, Q4Shape s) {
  pdl_launch();
  pdl_wait();
  const int G = s.G, D = s.D, d2 = D >> 1, ng = s.ng(), per = D >> 4;
  const size_t W = (size_t)(H + 2 * G) * D;
  const int kv = (G * ng * 8 + 31) / 32 * 32;  // whole warps: the shuffles are warp-wide
  const int items = kv + H * per, i = blockIdx.y * WRITE_THREADS + threadIdx.x;
  if (i < kv) {
    const int unit = i >> 3, g = unit / ng, gi = unit % ng;
    const int e = gi * Q4_GROUP + (i & 7) * 8;  // this lane's first element
    const bool mine = g < G && e < D;
    const bool first = e < d2;
    const int ec = first ? e : e - d2, partner = first ? e + d2 : e - d2;
    const uint32_t sign = first ? 0x80008000u : 0u;  // x c - y s in the first half of the row, x c + y s in the second
    // (The next row's loads are under way while this one is worked on: 23.9 us for 4352 rows, 25.1 without.)
    uint4 nx, ny, nv;
    int np, na;
    auto fetch = [&](int t) {
      np = na = -1;
      nx = ny = nv = make_uint4(0, 0, 0, 0);
      if (mine && t < T) {
        np = pos[t], na = slot[t];
        const __half* src = QKV + t * W + (size_t)(H + g) * D;
        nx = *reinterpret_cast<const uint4*>(src + e), ny = *reinterpret_cast<const uint4*>(src + partner);
        nv = *reinterpret_cast<const uint4*>(src + (size_t)G * D + e);
      }
    };
    fetch(blockIdx.x);
    for (int t = blockIdx.x; t < T; t += gridDim.x) {
      uint4 k = make_uint4(0, 0, 0, 0);
      const uint4 x = nx, y = ny, v = nv;
      const int p = np, at = na;
      fetch(t + gridDim.x);
      if (mine) {
        const bool in = p >= 0 && p < NPOS;
        const size_t to = (size_t)(in ? p : 0) * d2 + ec;
        uint64_t c[4], sn[4];
        load8(Ct + to, in, c);
        load8(St + to, in, sn);
        k.x = rotated(floats(x.x), c[0], floats(y.x ^ sign), sn[0]);
        k.y = rotated(floats(x.y), c[1], floats(y.y ^ sign), sn[1]);
        k.z = rotated(floats(x.z), c[2], floats(y.z ^ sign), sn[2]);
        k.w = rotated(floats(x.w), c[3], floats(y.w ^ sign), sn[3]);
        const size_t dd = ((size_t)t * G + g) * D + e;
        *reinterpret_cast<uint4*>(Kd + dd) = k;
        *reinterpret_cast<uint4*>(Vd + dd) = v;
      }
      uint32_t kw, kh, vw, vh;
      quantise8(k, kw, kh);
      quantise8(v, vw, vh);
      if (mine && at >= 0 && at < s.NP * s.P) {
        const int page = at / s.P, row = at - page * s.P;
        const size_t rec = ((size_t)page * G + g) * s.record(), code = rec + (size_t)row * d2 + (e >> 1);
        *reinterpret_cast<uint32_t*>(Kc + code) = kw;
        *reinterpret_cast<uint32_t*>(Vc + code) = vw;
        if ((i & 7) == 0) {
          const size_t h = rec + (size_t)s.P * d2 + 2 * (row * ng + gi);
          *reinterpret_cast<unsigned short*>(Kc + h) = (unsigned short)kh;
          *reinterpret_cast<unsigned short*>(Vc + h) = (unsigned short)vh;
        }
      }
    }
  } else if (i < items) {
    const int h = (i - kv) / per, ch = (i - kv) % per;
    const size_t from = (size_t)h * D + ch * 8;
#pragma unroll 2
    for (int t = blockIdx.x; t < T; t += gridDim.x) {
      const int p = pos[t];
      const bool in = p >= 0 && p < NPOS;
      const __half* src = QKV + t * W + from;
      const uint4 x1 = *reinterpret_cast<const uint4*>(src), x2 = *reinterpret_cast<const uint4*>(src + d2);
      const uint32_t a[4] = {x1.x, x1.y, x1.z, x1.w}, b[4] = {x2.x, x2.y, x2.z, x2.w};
      const size_t to = (size_t)(in ? p : 0) * d2 + ch * 8;
      uint64_t c[4], sn[4];
      load8(Ct + to, in, c);
      load8(St + to, in, sn);
      uint32_t y1[4], y2[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t u = floats(a[j]), w = floats(b[j]);
        y1[j] = rotated(u, c[j], floats(b[j] ^ 0x80008000u), sn[j]);
        y2[j] = rotated(w, c[j], u, sn[j]);
      }
      __half* dst = Q + (size_t)t * H * D + from;
      *reinterpret_cast<uint4*>(dst) = make_uint4(y1[0], y1[1], y1[2], y1[3]);
      *reinterpret_cast<uint4*>(dst + d2) = make_uint4(y2[0], y2[1], y2[2], y2[3]);
    }
  }
}

// Rows of the cache as f16 (exactly what they stand for); zeros for a slot outside the cache.
// A thread reads eight elements' codes and writes them as one 16-byte store; it keeps its place in the
// row and goes from row to row, four at a time in flight. HBM-bound: the f16 rows are four fifths of it
// (4352 rows of 8 heads, D 128: 7.6 us with its launch for 22.6 MB).
__global__ void __launch_bounds__(256)
    kv_unpack_q4_kernel(const unsigned char* __restrict__ Kc, const unsigned char* __restrict__ Vc, const int* __restrict__ slot,
                        __half* __restrict__ K, __half* __restrict__ V, int N, Q4Shape s, int rows) {
  pdl_launch();
  pdl_wait();
  const int per = s.D >> 3, G = s.G, ng = s.ng(), half = G * per, items = 2 * half;
  // `rows` rows side by side in a block where a row has fewer items than threads.
  const int r = threadIdx.x / (256 / rows), i = blockIdx.y * (256 / rows) + threadIdx.x % (256 / rows);
  if (i >= items) return;
  const bool isv = i >= half;
  const int j = isv ? i - half : i, g = j / per, ch = j % per;
  const unsigned char* cache = (isv ? Vc : Kc) + (size_t)g * s.record();
  __half* out = (isv ? V : K) + (size_t)g * s.D + ch * 8;
  const size_t page_bytes = (size_t)G * s.record();
  const int code = ch * 4, head = s.P * (s.D >> 1) + 2 * (ch >> 3);
  const int step = gridDim.x * rows;
  for (int n0 = blockIdx.x * rows + r; n0 < N; n0 += 4 * step) {
    int at[4];
    uint32_t w[4], hd[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = n0 + u * step < N ? slot[n0 + u * step] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      w[u] = hd[u] = 0;
      if (at[u] >= 0 && at[u] < s.NP * s.P) {
        const int page = at[u] / s.P, row = at[u] - page * s.P;
        const unsigned char* rec = cache + page * page_bytes;
        w[u] = *reinterpret_cast<const uint32_t*>(rec + code + (size_t)row * (s.D >> 1));
        hd[u] = *reinterpret_cast<const unsigned short*>(rec + head + 2 * row * ng);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (n0 + u * step >= N) break;
      // 1024 + code (64 + code: the upper nibbles of a byte weigh a sixteenth), less 1024 + z or 64 + z,
      // times the scale: exact at every step.
      const uint32_t z = hd[u] & 15u, sc = __byte_perm(hd[u] & 0xfff0u, 0, 0x1010);
      const uint32_t c0 = (z | z << 16) | 0xe400e400u, c1 = (z << 4 | z << 20) | 0xd400d400u, up = w[u] >> 8;
      uint32_t e[4] = {(w[u] & 0x000f000fu) | 0x64006400u, (w[u] & 0x00f000f0u) | 0x64006400u, (up & 0x000f000fu) | 0x64006400u,
                       (up & 0x00f000f0u) | 0x64006400u};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2 x = *reinterpret_cast<__half2*>(&e[j]);
        const __half2 d = (j & 1) ? __hfma2(x, __float2half2_rn(0.0625f), *reinterpret_cast<const __half2*>(&c1))
                                  : __hadd2(x, *reinterpret_cast<const __half2*>(&c0));
        const __half2 y = __hmul2(d, *reinterpret_cast<const __half2*>(&sc));
        e[j] = *reinterpret_cast<const uint32_t*>(&y);
      }
      *reinterpret_cast<uint4*>(out + (size_t)(n0 + u * step) * G * s.D) = make_uint4(e[0], e[1], e[2], e[3]);
    }
  }
}

// Attention of one query row and head over its first `n` cached tokens, by one warp, for any page
// size and head_dim: a key at a time, an f32 online softmax. A lane owns the elements of words
// lane, lane + 32, ... that is, at most one word of eight (D <= 256).
// Tokens beyond the block table lie on page 0 (as decode_attention reads them); a page outside the
// cache reads as zeros.
__device__ __forceinline__ void attend_q4(const __half* __restrict__ q, const unsigned char* __restrict__ Kc,
                                          const unsigned char* __restrict__ Vc, const int* __restrict__ row, int MP,
                                          long long n, int g, float scale, const Q4Shape& s, __half* __restrict__ o) {
  const int lane = threadIdx.x & 31, words = s.D >> 3, ng = s.ng();
  const bool mine = lane < words;
  float qv[8], acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    qv[e] = mine ? __half2float(q[lane * 8 + e]) : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (long long t = 0; t < n; ++t) {
    const long long col = t / s.P;
    const int at = (int)(t % s.P), page = col < MP ? row[col] : 0;
    const bool in = mine && page >= 0 && page < s.NP;
    const size_t rec = ((size_t)(in ? page : 0) * s.G + g) * s.record();
    const size_t cw = rec + (size_t)at * (s.D >> 1) + lane * 4, hw = rec + (size_t)s.P * (s.D >> 1) + 2 * (at * ng + (lane >> 3));
    float x = 0.f, v[8];
    uint32_t vw = 0;
    float vs = 0.f, vz = 0.f;
    if (in) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(Kc + cw);
      const uint32_t head = *reinterpret_cast<const unsigned short*>(Kc + hw);
      const float zp = q4_zero(head);
#pragma unroll
      for (int e = 0; e < 8; ++e) x += ((float)q4_code(w, e) - zp) * qv[e];
      x *= q4_scale(head);
      vw = *reinterpret_cast<const uint32_t*>(Vc + cw);
      const uint32_t vh = *reinterpret_cast<const unsigned short*>(Vc + hw);
      vs = q4_scale(vh), vz = q4_zero(vh);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = vs * ((float)q4_code(vw, e) - vz);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    x *= scale;
    const float m2 = fmaxf(m, x), a = expf(m - m2), p = expf(x - m2);
    l = l * a + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * a + p * v[e];
    m = m2;
  }
  if (mine) {
    uint4 y;  // n == 0: 0/0, NaN
    y.x = pack_h2(acc[0] / l, acc[1] / l), y.y = pack_h2(acc[2] / l, acc[3] / l);
    y.z = pack_h2(acc[4] / l, acc[5] / l), y.w = pack_h2(acc[6] / l, acc[7] / l);
    *reinterpret_cast<uint4*>(o + lane * 8) = y;
  }
}

__global__ void decode_q4_generic_kernel(const __half* __restrict__ Q, const unsigned char* __restrict__ Kc,
                                         const unsigned char* __restrict__ Vc, const int* __restrict__ table,
                                         const int* __restrict__ lens, __half* __restrict__ O, float scale, int B, int H,
                                         int MP, Q4Shape s) {
  pdl_launch();
  pdl_wait();
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= (long long)B * H) return;
  const int b = (int)(w / H), h = (int)(w % H);
  attend_q4(Q + w * s.D, Kc, Vc, table + (size_t)b * MP, MP, lens[b], h / (H / s.G), scale, s, O + w * s.D);
}

__global__ void chunk_q4_generic_kernel(const __half* __restrict__ Q, const unsigned char* __restrict__ Kc,
                                        const unsigned char* __restrict__ Vc, const int* __restrict__ table,
                                        const int* __restrict__ meta, __half* __restrict__ O, float scale, int T, int H,
                                        int MP, Q4Shape s) {
  pdl_launch();
  pdl_wait();
  const int* m = meta + 4 * blockIdx.y;
  const int row0 = m[0], nrows = m[1], pos0 = m[2];
  if (row0 < 0 || nrows <= 0 || pos0 < 0 || nrows > T - row0) return;  // a descriptor outside the step is skipped
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= (long long)nrows * H) return;
  const int r = (int)(w / H), h = (int)(w % H);
  const size_t at = ((size_t)(row0 + r) * H + h) * s.D;
  attend_q4(Q + at, Kc, Vc, table + (size_t)row0 * MP, MP, (long long)pos0 + r + 1, h / (H / s.G), scale, s, O + at);
}

// For every cache a and pair n: page pairs[n][1] of caches[a] = page pairs[n][0]. One block per
// (pair, cache) at a time; a thread has eight 16-byte loads in flight before its first store (448 pages of 32 KB:
// 5.3 us, 8.4 with a load and a store in turn; 12160 of them: 126 us, 0.97 of the copy rate. HBM-bound).
constexpr int PAGE_THREADS = 256;

__global__ void __launch_bounds__(PAGE_THREADS) page_copy_kernel(const unsigned long long* __restrict__ caches, const int* __restrict__ pairs, int A,
                                 int n, int NP, int words) {
  pdl_launch();
  pdl_wait();
  const long long jobs = (long long)n * A;
  for (long long j = blockIdx.x; j < jobs; j += gridDim.x) {
    const int pair = (int)(j / A), a = (int)(j % A);
    const int src = pairs[2 * pair], dst = pairs[2 * pair + 1];
    const unsigned long long cache = caches[a];
    if (src < 0 || src >= NP || dst < 0 || dst >= NP || src == dst || cache == 0 || cache % 16) continue;
    const uint4* from = (const uint4*)cache + (size_t)src * words;
    uint4* to = (uint4*)cache + (size_t)dst * words;
    for (int i = threadIdx.x; i < words; i += 8 * PAGE_THREADS) {
      uint4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * PAGE_THREADS < words) v[u] = from[i + u * PAGE_THREADS];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * PAGE_THREADS < words) to[i + u * PAGE_THREADS] = v[u];
    }
  }
}

// Blocks along the rows, when `y` blocks share a row: one per row, at most `cap` in all.
unsigned rows_for(int rows, unsigned y, int cap) {
  const unsigned most = (unsigned)cap / y > 0 ? (unsigned)cap / y : 1u;
  return (unsigned)rows < most ? (unsigned)rows : most;
}

}  // namespace

int make_kv_q4(Ctx* c, Op& op) {
  const auto& s = op.shapes;
  auto bad = [&](const char* why) { return fail(c, op.name + ": " + why); };
  for (const auto& a : s)
    for (int64_t d : a)
      if (d > 0x40000000LL) return bad("a dimension is beyond 2^30");  // (loops step past the last row in 32 bits)
  Q4Shape q;
  const char* why = nullptr;
  switch (op.kind) {
    case K_ROPE_KV_Q4: {
      // QKV[T,W], pos[T], slot[T], C, S [NPOS,D/2], Q[T,H,D], Kc, Vc, K, V [T,G,D]
      if (s[0].size() != 2 || s[1].size() != 1 || s[2].size() != 1 || s[3].size() != 2 || s[4] != s[3] || s[5].size() != 3 ||
          s[8].size() != 3 || s[9] != s[8])
        return bad("shapes are QKV[T,W], pos[T], slot[T], C, S[NPOS,D/2], Q[T,H,D], Kc, Vc, K, V[T,G,D]");
      const int64_t T = s[0][0], H = s[5][1], D = s[5][2];
      if ((why = q4_shape(op, 6, D, &q))) return bad(why);
      if (s[1][0] != T || s[2][0] != T || s[5][0] != T || s[8][0] != T) return bad("QKV, pos, slot, Q, K and V have T rows");
      if (s[3][1] != D / 2) return bad("the rotation tables are [NPOS, D/2]");
      if (s[8][1] != q.G || s[8][2] != D) return bad("K and V are [T,G,D]");
      if (s[0][1] != (H + 2 * q.G) * D) return bad("W must be (H + 2G) * D");
      return 0;
    }
    case K_KV_UNPACK_Q4:
      if (s[2].size() != 1 || s[3].size() != 3 || s[4] != s[3] || s[3][0] != s[2][0])
        return bad("shapes are Kc, Vc, slot[N], K, V[N,G,D]");
      if ((why = q4_shape(op, 0, s[3][2], &q))) return bad(why);
      if (s[3][1] != q.G) return bad("K and V are [N,G,D]");
      return 0;
    case K_DECODE_ATTENTION_Q4:
    case K_CHUNK_ATTENTION_Q4: {
      const bool chunk = op.kind == K_CHUNK_ATTENTION_Q4;
      const char* shapes = chunk ? "shapes are Q[T,H,D], Kc, Vc, table[T,MP], meta[C,4], O[T,H,D]"
                                 : "shapes are Q[B,H,D], Kc, Vc, table[B,MP], lens[B], O[B,H,D]";
      if (s[0].size() != 3 || s[5] != s[0] || s[3].size() != 2 || s[3][0] != s[0][0]) return bad(shapes);
      if (chunk ? s[4].size() != 2 || s[4][1] != 4 : s[4].size() != 1 || s[4][0] != s[0][0]) return bad(shapes);
      if ((why = q4_shape(op, 1, s[0][2], &q))) return bad(why);
      if (s[0][1] < 1 || s[0][1] % q.G) return bad("heads must be a multiple of kv heads");
      if (chunk && s[4][0] > 65535) return bad("at most 65535 chunks");
      const int T = (int)s[0][0], H = (int)s[0][1], MP = (int)s[3][1];
      op.p0 = chunk ? chunk_q4_takes(q, T, H, (int)s[4][0], MP) : decode_q4_takes(q, T, MP);
      if (!op.p0) return 0;
      if (void** work = &c->q4_work[q.D == 128]; !*work) {
        const size_t d = decode_q4_workspace(c, q.D), k = chunk_q4_workspace(c, q.D);
        TB_CUDA(c, cudaMalloc(work, d > k ? d : k));
      }
      return chunk ? make_chunk_q4(c, op, q) : make_decode_q4(c, op, q);
    }
    case K_PAGE_COPY:
      if (s[0].size() != 1 || s[1].size() != 2 || s[1][1] != 2) return bad("shapes are caches i64[A], pairs[N,2]");
      return 0;
    default:
      return bad("not a 4-bit cache kernel");
  }
}

int launch_kv_q4(Ctx* c, Op& op, const uint64_t* a) {
  const auto& s = op.shapes;
  auto bad = [&](const char* why) { return fail(c, op.name + ": " + why); };
  Q4Shape q;
  TB_CUDA(c, cudaSetDevice(c->device));  // the caller's thread may have another device current
  switch (op.kind) {
    case K_ROPE_KV_Q4: {
      const int T = (int)s[0][0], H = (int)s[5][1], D = (int)s[5][2], NPOS = (int)s[3][0];
      q4_shape(op, 6, D, &q);
      if (T == 0) return 0;
      for (int i : {0, 5, 6, 7, 8, 9})
        if (!aligned_to(a[i], 16)) return bad("QKV, Q, K, V and the caches must be 16-byte aligned");
      const int items = (q.G * q.ng() * 8 + 31) / 32 * 32 + H * (D / 16);
      for (int i : {3, 4})
        if (!aligned_to(a[i], 16)) return bad("the rotation tables must be 16-byte aligned");
      if (!aligned_to(a[1] | a[2], 4)) return bad("pos and slot must be 4-byte aligned");
      const unsigned y = (unsigned)((items + WRITE_THREADS - 1) / WRITE_THREADS);
      TB_CUDA(c, launch_k(c, rope_kv_q4_kernel, dim3(rows_for(T, y, c->sm_count * 16), y), dim3(WRITE_THREADS), 0, 1, (const __half*)a[0],
                          (const int*)a[1], (const int*)a[2], (const float*)a[3], (const float*)a[4], (__half*)a[5],
                          (unsigned char*)a[6], (unsigned char*)a[7], (__half*)a[8], (__half*)a[9], T, H, NPOS, q));
      break;
    }
    case K_KV_UNPACK_Q4: {
      const int N = (int)s[2][0], D = (int)s[3][2];
      q4_shape(op, 0, D, &q);
      if (N == 0) return 0;
      for (int i : {0, 1, 3, 4})
        if (!aligned_to(a[i], 16)) return bad("K, V and the caches must be 16-byte aligned");
      if (!aligned_to(a[2], 4)) return bad("slot must be 4-byte aligned");
      const int items = 2 * q.G * (D / 8);
      int rows = 1;
      while (rows < 16 && items * rows * 2 <= 256) rows *= 2;
      const unsigned y = (unsigned)((items + 256 / rows - 1) / (256 / rows));
      TB_CUDA(c, launch_k(c, kv_unpack_q4_kernel, dim3(rows_for((N + rows - 1) / rows, y, c->sm_count * 8), y), dim3(256), 0, 1,
                          (const unsigned char*)a[0], (const unsigned char*)a[1], (const int*)a[2], (__half*)a[3],
                          (__half*)a[4], N, q, rows));
      break;
    }
    case K_DECODE_ATTENTION_Q4:
    case K_CHUNK_ATTENTION_Q4: {
      const int T = (int)s[0][0], H = (int)s[0][1], D = (int)s[0][2], MP = (int)s[3][1];
      q4_shape(op, 1, D, &q);
      for (int i : {0, 1, 2, 5})
        if (!aligned_to(a[i], 16)) return bad("Q, O and the caches must be 16-byte aligned");
      if (op.kind == K_CHUNK_ATTENTION_Q4 && !aligned_to(a[4], 16)) return bad("meta must be 16-byte aligned");
      if (!aligned_to(a[3] | a[4], 4)) return bad("the block table and lens must be 4-byte aligned");
      const unsigned blocks = (unsigned)(((long long)T * H + 3) / 4);
      if (T == 0) return 0;
      if (op.p0 && op.kind == K_DECODE_ATTENTION_Q4) return launch_decode_q4(c, op, a, q);
      // (The tensor-core kernel masks before it scales, and takes the maximum of the unscaled scores.)
      if (op.p0 && bits_f32(a[6]) > 0.f && bits_f32(a[6]) < INFINITY) return launch_chunk_q4(c, op, a, q);
      if (op.kind == K_DECODE_ATTENTION_Q4) {
        TB_CUDA(c, launch_k(c, decode_q4_generic_kernel, dim3(blocks), dim3(128), 0, 1, (const __half*)a[0],
                            (const unsigned char*)a[1], (const unsigned char*)a[2], (const int*)a[3], (const int*)a[4],
                            (__half*)a[5], bits_f32(a[6]), T, H, MP, q));
      } else {
        if (s[4][0] == 0) return 0;
        TB_CUDA(c, launch_k(c, chunk_q4_generic_kernel, dim3(blocks, (unsigned)s[4][0]), dim3(128), 0, 1,
                            (const __half*)a[0], (const unsigned char*)a[1], (const unsigned char*)a[2], (const int*)a[3],
                            (const int*)a[4], (__half*)a[5], bits_f32(a[6]), T, H, MP, q));
      }
      break;
    }
    case K_PAGE_COPY: {
      const int A = (int)s[0][0], n = (int)(uint32_t)a[2], NP = (int)(uint32_t)a[3], bytes = (int)(uint32_t)a[4];
      if (n < 0 || n > s[1][0]) return bad("0 <= n <= N pairs");
      if (NP < 0 || bytes < 16 || bytes % 16) return bad("the page size must be a positive multiple of 16 bytes, NP not negative");
      if (!aligned_to(a[0], 8) || !aligned_to(a[1], 4)) return bad("the address table must be 8-byte aligned");
      if (A == 0 || n == 0) return 0;
      const long long jobs = (long long)A * n, cap = (long long)c->sm_count * 8;
      TB_CUDA(c, launch_k(c, page_copy_kernel, dim3((unsigned)(jobs < cap ? jobs : cap)), dim3(PAGE_THREADS), 0, 1,
                          (const unsigned long long*)a[0], (const int*)a[1], A, n, NP, bytes / 16));
      break;
    }
    default:
      return bad("not a 4-bit cache kernel");
  }
  c->launches += 1;
  TB_CUDA(c, cudaGetLastError());
  return 0;
}

}  // namespace tb
