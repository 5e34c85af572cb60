// Cache pages of 8- and 4-bit integers: rows quantised as they are written, and read back as bf16.
//
// 64 channels of one token and head form a group with the scale  s = bf16(max|x| / m),  m = 127 or 7,
// and the codes  c = round(x * (1 / s)) in [-m, m]  (products and the reciprocal in FP32, halves to even);
// a value is read back as bf16(c * s).  The scale is rounded before it is used, so its rounding costs
// nothing: only the grid moves by it.  bf16 rather than FP32 scales keep a 4-bit row of 128 channels at
// 68 bytes instead of 72; bf16 rather than FP16 so that every finite input has one.  A group whose largest
// magnitude is under m 2^-100 is stored as zeros (its reciprocal would overflow), a group that holds an
// infinity or a NaN gets a NaN scale and reads back as NaN.
//
// A prefix that many sequences share is expanded for the tensor unit (scored_flash_tc05.cu) as FP16: code * s / 2^e with e
// the exponent of the largest scale of the prefix and head, at most 254 and rounded by 2^-11 (bf16 would round
// every key by 2^-8 again, which a capped model's scores of some tens turn into percents of a weight).
//
// Writing and reading are bound by memory.  A thread has one column of 8 channels (16 bytes of bf16) in the rows of its
// block, so what depends on the column is computed once, and loads of several rows are in flight; the rows' places are looked
// up once a block.  (A division of 64 bits a piece more than doubled the time of a write; 16 channels a thread, which leave
// sectors half written, made reading a quarter slower.)  8,168 rows of 4 heads of 128 channels are written in 7.6 us as 8 bits
// (25.4 MB in and out, 0.52 of a copy's rate) and in 7.9 as 4 bits (21.2 MB, 0.42): two rows' loads are in flight a thread, and
// the shuffles wait for them.  41,394 are read in 30.1 us (128.5 MB, 0.66) and in 22.4 (107.3 MB, 0.74): a block waits for its
// places before its first load.
#include "include/us_common.cuh"

namespace {

struct WriteArgs {
  const __nv_bfloat16 *k, *v;
  const void* slots;           // int32 or int64 [rows]; negative: the row is not written
  uint8_t *kc, *vc;            // [pages, page, heads, dim * bits / 8]
  __nv_bfloat16 *ks, *vs;      // [pages, heads, page, dim / 64]
  long long ldk, hsk, ldv, hsv;   // elements between rows and between heads
  long long capacity;          // pages * page
  int rows, page, heads, dim, wide;
  unsigned int* status;
};

__device__ __forceinline__ float small_int(uint32_t u, float offset) {   // u in [0, 2^22)
  return __uint_as_float(0x4B000000u | u) - (8388608.f + offset);
}

template <int BITS>
__device__ __forceinline__ void quantise8(const uint4& raw, uint32_t (&code)[2], __nv_bfloat16& scale) {
  constexpr float kMost = BITS == 8 ? 127.f : 7.f;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t top = 0;            // magnitudes as 15-bit integers: NaN above infinity above every number
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  top = max(top & 0xffffu, top >> 16);
  const float most = __uint_as_float(top << 16);
  float inv = 0.f;
  scale = us::f2bf(0.f);
  if (top >= 0x7f80u) {
    scale = __ushort_as_bfloat16(0x7fffu);
  } else if (most >= kMost * 0x1p-100f) {
    scale = us::f2bf(__fdiv_rn(most, kMost));
    inv = __frcp_rn(us::bf2f(scale));
  }
  // 1.5 * 2^23 + c: the rounded integer in the low mantissa bits (halves to even, as the sum is rounded).  The product is
  // rounded before the sum, as in the definition: no fused multiply-add.  It stays under m + 1 / 2 without a clamp: the
  // scale is at least 1 - 2^-8 of max|x| / m, and m / (1 - 2^-8) is 127.498 or 7.03.
  uint32_t t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = __uint_as_float(i & 1 ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    t[i] = __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f + (BITS == 4 ? 8.f : 0.f)));
  }
  const bool fine = top < 0x7f80u;
  if constexpr (BITS == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t c = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
      code[i] = fine ? c : 0u;
    }
  } else {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) c |= (t[i] & 15u) << (4 * i);
    code[0] = fine ? c : 0x88888888u;
    code[1] = 0;
  }
}

constexpr int kWriteRows = 8;

template <int BITS>
__global__ void __launch_bounds__(256) quant_write_kernel(const WriteArgs a) {
  US_PDL_PROLOGUE();
  const int per_row = a.heads * (a.dim >> 3), block_row = blockIdx.x * kWriteRows;
  const int together = max(1, 256 / per_row);            // rows that the block's threads stand on
  const int r0 = (int)threadIdx.x / per_row, c0 = (int)threadIdx.x - r0 * per_row;
  // (eight threads of a group are on one row: rows have a multiple of eight pieces.  Threads past the last row or column
  // take part in the shuffles on ones that are there, and write nothing.)
  for (int first = 0; first < per_row; first += 256) {
    const bool mine = r0 < together && first + c0 < per_row;
    const int c = mine ? first + c0 : c0 & 7;
    const int head = (c << 3) / a.dim, ch = (c << 3) - head * a.dim;
    const __nv_bfloat16 *k = a.k + head * a.hsk + ch, *v = a.v + head * a.hsv + ch;
    const uint32_t byte = head * (a.dim * BITS / 8) + ch * BITS / 8, row_bytes = a.heads * (a.dim * BITS / 8);
    const uint32_t group = (uint32_t)head * a.page;
#pragma unroll 2
    for (int i = 0; i < kWriteRows; i += together) {
      const int row = block_row + i + r0, from = min(row, a.rows - 1);
      const uint4 rk = *reinterpret_cast<const uint4*>(k + from * a.ldk);
      const uint4 rv = *reinterpret_cast<const uint4*>(v + from * a.ldv);
      const long long slot = a.wide ? ((const long long*)a.slots)[from] : (long long)((const int*)a.slots)[from];
      uint32_t ck[2], cv[2];
      __nv_bfloat16 sk, sv;
      quantise8<BITS>(rk, ck, sk);
      quantise8<BITS>(rv, cv, sv);
      if (!mine || i + r0 >= kWriteRows || row >= a.rows || slot < 0) continue;
      if (slot >= a.capacity) {
        us_dev_fail(a.status, US_DEV_BOUNDS);
        continue;
      }
      const unsigned long long to = (unsigned long long)(uint32_t)slot * row_bytes + byte;
      if constexpr (BITS == 8) {
        *reinterpret_cast<uint2*>(a.kc + to) = make_uint2(ck[0], ck[1]);
        *reinterpret_cast<uint2*>(a.vc + to) = make_uint2(cv[0], cv[1]);
      } else {
        *reinterpret_cast<uint32_t*>(a.kc + to) = ck[0];
        *reinterpret_cast<uint32_t*>(a.vc + to) = cv[0];
      }
      if ((ch & 63) == 0) {
        const uint32_t p = (uint32_t)slot / (uint32_t)a.page, off = (uint32_t)slot - p * (uint32_t)a.page;
        const unsigned long long s = ((unsigned long long)p * (uint32_t)(a.heads * a.page) + group + off) * (uint32_t)(a.dim >> 6) + (ch >> 6);
        a.ks[s] = sk;
        a.vs[s] = sv;
      }
    }
  }
}

struct ReadArgs {
  const uint8_t *kc, *vc;
  const __nv_bfloat16 *ks, *vs;
  const int *table, *cu, *out_cu;
  __nv_bfloat16 *ko, *vo;
  long long ldo;
  int B, max_pages, pages, page, heads, dim, total, out_rows;
  unsigned int* status;
};

constexpr int kReadRows = 16;

__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t mul_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Eight codes under a scale as bf16, two at a time: a code is a bf16 number exactly (128 + its low bits, less 128 or 256,
// or 136), and one product of two bf16 numbers, rounded once, is the definition's value.
template <int BITS>
struct Code {
  typedef uint2 type;
};
template <>
struct Code<4> {
  typedef uint32_t type;
};
template <int BITS>
__device__ __forceinline__ void expand8(const typename Code<BITS>::type& raw, uint32_t scale2, uint4& out) {
  uint32_t o[4];
  if constexpr (BITS == 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = __byte_perm(j < 2 ? raw.x : raw.y, 0, j & 1 ? 0x4342 : 0x4140);
      o[j] = mul_bf2(sub_bf2((x & 0x007f007fu) | 0x43004300u, (x & 0x00800080u) | 0x43004300u), scale2);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = __byte_perm(raw, 0, 0x4440 + j) * 4097u;      // a byte's nibbles in the low bits of both halves
      o[j] = mul_bf2(sub_bf2((x & 0x000f000fu) | 0x43004300u, 0x43084308u), scale2);
    }
  }
  out = make_uint4(o[0], o[1], o[2], o[3]);
}
template <int BITS, int ROWS>
__global__ void __launch_bounds__(256) quant_gather_kernel(const ReadArgs a) {
  US_PDL_PROLOGUE();
  __shared__ long long src[ROWS], at[ROWS], dst[ROWS];   // first byte (-1: a page outside the cache), first scale of head 0,
                                                         // first output (-1: none) of a row
  const int r0 = blockIdx.x * ROWS;
  if (threadIdx.x < ROWS) {
    const int r = r0 + threadIdx.x;
    long long s = -1, w = 0, d = -1;
    if (r >= a.cu[0] && r < min(a.total, a.cu[a.B])) {
      int lo = 0, hi = a.B - 1;                 // sequence of packed row r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= r) lo = mid; else hi = mid - 1;
      }
      const int pos = r - a.cu[lo], pi = pos / a.page;
      const int pg = pi < a.max_pages ? a.table[(long long)lo * a.max_pages + pi] : -1;
      const int to = (a.out_cu ? a.out_cu[lo] : a.cu[lo]) + pos;
      d = to * a.ldo;
      if (to < 0 || to >= a.out_rows) {
        d = -1;
        us_dev_fail(a.status, US_DEV_BOUNDS);
      }
      if (pg >= 0 && pg < a.pages) {
        s = ((long long)pg * a.page + (pos - pi * a.page)) * a.heads * (a.dim * BITS / 8);
        w = ((long long)pg * a.heads * a.page + (pos - pi * a.page)) * (a.dim >> 6);
      } else {
        us_dev_fail(a.status, US_DEV_BOUNDS);
      }
    }
    src[threadIdx.x] = s;
    dst[threadIdx.x] = d;
    at[threadIdx.x] = w;
  }
  if (r0 == 0 && threadIdx.x == ROWS && a.cu[a.B] > a.total) us_dev_fail(a.status, US_DEV_BOUNDS);      // rows left out
  __syncthreads();
  const int per_row = a.heads * (a.dim >> 3), groups = a.dim >> 6;
  const int together = max(1, 256 / per_row);            // rows that the block's threads stand on
  const int t0 = (int)threadIdx.x / per_row;
  if (t0 >= together) return;
  for (int c = (int)threadIdx.x - t0 * per_row; c < per_row; c += 256) {
    const int head = (c << 3) / a.dim, ch = (c << 3) - head * a.dim;
    const int byte = head * (a.dim * BITS / 8) + ch * BITS / 8, sc = head * a.page * groups + (ch >> 6);
    const uint8_t *kc = a.kc + byte, *vc = a.vc + byte;
    const unsigned short *ks = reinterpret_cast<const unsigned short*>(a.ks) + sc, *vs = reinterpret_cast<const unsigned short*>(a.vs) + sc;
    __nv_bfloat16 *ko = a.ko + (c << 3), *vo = a.vo + (c << 3);
    for (int i0 = t0; i0 < ROWS; i0 += 4 * together) {     // the loads of four rows, then their values
      typename Code<BITS>::type k[4], v[4];
      uint32_t s[4], t[4];
      long long d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * together;
        d[j] = i < ROWS ? dst[i] : -1;
        const long long from = i < ROWS ? src[i] : -1, w = i < ROWS ? at[i] : 0;
        s[j] = t[j] = 0;
        k[j] = v[j] = typename Code<BITS>::type{};
        if (from >= 0) {
          k[j] = *reinterpret_cast<const typename Code<BITS>::type*>(kc + from);
          v[j] = *reinterpret_cast<const typename Code<BITS>::type*>(vc + from);
          s[j] = ks[w];
          t[j] = vs[w];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (d[j] < 0) continue;
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        expand8<BITS>(k[j], s[j] * 65537u, x);
        expand8<BITS>(v[j], t[j] * 65537u, y);
        *reinterpret_cast<uint4*>(ko + d[j]) = x;
        *reinterpret_cast<uint4*>(vo + d[j]) = y;
      }
    }
  }
}

struct PrefixArgs {
  const uint8_t *kc, *vc;
  const __nv_bfloat16 *ks, *vs;
  const int *table, *cu_rows, *shared;
  const __nv_bfloat16* q;
  long long ldq;
  __half *ko, *vo, *qo;        // [groups][max_len][heads][dim] twice, [B][Hq][dim]
  float* q_back;               // [B * Hq]: what a row's scores are multiplied by
  int2* exps;                  // [groups * heads]: exponent fields of the largest scale of K and of V
  int groups, max_len, max_pages, pages, page, heads, dim, batch, Hq;
  unsigned int* status;
};

__device__ __forceinline__ float power_of_two(int field) { return __uint_as_float((uint32_t)min(max(field, 0), 254) << 23); }
// rows of a group's prefix; a longer one than the host was told ends there
__device__ __forceinline__ int prefix_rows(const PrefixArgs& a, int g) {
  if (a.cu_rows[g + 1] <= a.cu_rows[g] || (unsigned)a.cu_rows[g] >= (unsigned)a.batch) return 0;
  if (a.shared[g] > a.max_len) us_dev_fail(a.status, US_DEV_BOUNDS);
  return min(a.shared[g], a.max_len);
}
// slot of position `pos` of a group's prefix, or -1
__device__ __forceinline__ long long prefix_slot(const PrefixArgs& a, int g, int pos) {
  const int pi = pos / a.page;
  const int pg = pi < a.max_pages ? a.table[(long long)a.cu_rows[g] * a.max_pages + pi] : -1;
  if (pg >= 0 && pg < a.pages) return (long long)pg * a.page + (pos - pi * a.page);
  us_dev_fail(a.status, US_DEV_BOUNDS);
  return -1;
}

// Blocks [0, groups * heads): the largest scales of a group's head.  The others: 16 rows of Q each, divided by the power of
// two of their largest channel.
__global__ void __launch_bounds__(512) prefix_scales_kernel(const PrefixArgs a) {
  US_PDL_PROLOGUE();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x < a.groups * a.heads) {
    __shared__ uint32_t most[2][16];
    const int g = blockIdx.x / a.heads, head = blockIdx.x - g * a.heads, groups = a.dim >> 6;
    const int len = prefix_rows(a, g);
    uint32_t k = 0, v = 0;
#pragma unroll 4
    for (int pos = threadIdx.x; pos < len; pos += 512) {
      const long long slot = prefix_slot(a, g, pos);
      if (slot < 0) continue;
      const long long p = slot / a.page, at = ((p * a.heads + head) * a.page + (slot - p * a.page)) * groups;
      for (int i = 0; i < groups; ++i) {
        const uint32_t x = (uint32_t)__bfloat16_as_ushort(a.ks[at + i]) & 0x7fffu, y = (uint32_t)__bfloat16_as_ushort(a.vs[at + i]) & 0x7fffu;
        k = max(k, x < 0x7f80u ? x : 0u);      // (of those that are numbers: the others lose their own group, not the prefix)
        v = max(v, y < 0x7f80u ? y : 0u);
      }
    }
    k = __reduce_max_sync(0xffffffffu, k);
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) {
      most[0][warp] = k;
      most[1][warp] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 16; ++i) {
        k = max(k, most[0][i]);
        v = max(v, most[1][i]);
      }
      a.exps[blockIdx.x] = make_int2((int)(k >> 7), (int)(v >> 7));
    }
    return;
  }
  const int row = ((int)blockIdx.x - a.groups * a.heads) * 16 + warp;
  if (row >= a.batch * a.Hq) return;
  const int b = row / a.Hq;
  const __nv_bfloat16* from = a.q + (long long)b * a.ldq + (long long)(row - b * a.Hq) * a.dim;
  uint32_t most = 0;
  for (int i = lane; i < a.dim; i += 32) most = max(most, (uint32_t)__bfloat16_as_ushort(from[i]) & 0x7fffu);
  most = __reduce_max_sync(0xffffffffu, most);
  const int e = min(max((int)(most >> 7), 1), 253);       // (the ends of the range beside the ones that have a reciprocal)
  const float down = power_of_two(254 - e);
  for (int i = lane; i < a.dim; i += 32) a.qo[(long long)row * a.dim + i] = __float2half_rn(us::bf2f(from[i]) * down);
  if (lane == 0) a.q_back[row] = power_of_two(e);
}

template <int BITS>
__global__ void __launch_bounds__(256) prefix_expand_kernel(const PrefixArgs a) {
  US_PDL_PROLOGUE();
  const int g = blockIdx.y, r0 = blockIdx.x * kReadRows;
  const int len = prefix_rows(a, g);
  if (r0 >= len) return;
  __shared__ long long src[kReadRows];
  if (threadIdx.x < kReadRows) src[threadIdx.x] = r0 + (int)threadIdx.x < len ? prefix_slot(a, g, r0 + threadIdx.x) : -1;
  __syncthreads();
  const bool plane_v = blockIdx.z != 0;
  const int per_head = a.dim >> 4, per_row = a.heads * per_head, groups = a.dim >> 6;
  const uint8_t* cache = plane_v ? a.vc : a.kc;
  const __nv_bfloat16* scales = plane_v ? a.vs : a.ks;
  __half* out = (plane_v ? a.vo : a.ko) + ((long long)g * a.max_len + r0) * a.heads * a.dim;
#pragma unroll 4
  for (int e = threadIdx.x; e < min(kReadRows, len - r0) * per_row; e += 256) {
    const int i = e / per_row, rest = e - i * per_row, head = rest / per_head, ch = (rest - head * per_head) * 16;
    uint4* to = reinterpret_cast<uint4*>(out + ((long long)i * a.heads + head) * a.dim + ch);
    const long long slot = src[i];
    if (slot < 0) {
      to[0] = to[1] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const int2 top = a.exps[g * a.heads + head];
    const long long p = slot / a.page;
    const float sc = us::bf2f(scales[((p * a.heads + head) * a.page + (slot - p * a.page)) * groups + (ch >> 6)]) *
                     power_of_two(254 - (plane_v ? top.y : top.x));
    const uint8_t* c = cache + (slot * a.heads + head) * (a.dim * BITS / 8) + ch * BITS / 8;
    uint32_t o[8];
    if constexpr (BITS == 8) {
      const uint4 raw = *reinterpret_cast<const uint4*>(c);
      const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t u = w[j >> 1] >> (16 * (j & 1));
        const __half2 b = __floats2half2_rn(small_int(u & 255u, 128.f) * sc, small_int((u >> 8) & 255u, 128.f) * sc);
        o[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t u = (j < 4 ? raw.x : raw.y) >> (8 * (j & 3));
        const __half2 b = __floats2half2_rn(small_int(u & 15u, 8.f) * sc, small_int((u >> 4) & 15u, 8.f) * sc);
        o[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    to[0] = make_uint4(o[0], o[1], o[2], o[3]);
    to[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

}  // namespace

// Rows k, v [rows, heads, dim] (bf16; row and head strides in elements, multiples of 8) into integer pages at
// `slots` (page * page_size + offset; int32, or int64 with wide != 0).  The slots of a call are distinct.
US_API int us_quant_write(const void* k, const void* v, long long ldk, long long hsk, long long ldv, long long hsv,
                          const void* slots, int wide, void* kc, void* vc, void* ks, void* vs, int rows, int pages,
                          int page, int heads, int dim, int bits, void* stream_) {
  US_REQUIRE(rows >= 0 && pages >= 1 && page >= 1 && heads >= 1 && dim >= 64 && dim % 64 == 0 && (bits == 8 || bits == 4));
  if (rows == 0) return US_OK;
  US_REQUIRE(k && v && slots && kc && vc && ks && vs);
  US_REQUIRE(((ldk | hsk | ldv | hsv) % 8) == 0 && aligned16(k) && aligned16(v) && aligned16(kc) && aligned16(vc));
  const WriteArgs a{(const __nv_bfloat16*)k, (const __nv_bfloat16*)v, slots, (uint8_t*)kc, (uint8_t*)vc,
                    (__nv_bfloat16*)ks, (__nv_bfloat16*)vs, ldk, hsk, ldv, hsv, (long long)pages * page, rows, page,
                    heads, dim, wide, us_status_ptr()};
  if ((long long)pages * page > 0x7fffffffLL) return US_ERR_LIMIT;
  US_CUDA_CHECK(us::launch_pdl(bits == 8 ? quant_write_kernel<8> : quant_write_kernel<4>, dim3((rows + kWriteRows - 1) / kWriteRows),
                               dim3(256), 0, (cudaStream_t)stream_, a));
  return US_OK;
}

// The first cu[s + 1] - cu[s] cached rows of every sequence as bf16 rows [total, heads, dim] (row pitch ldo), packed,
// or from row out_cu[s] on.  Rows past cu[B] are not written; a page outside the cache is read as zeros and sets the status word, as
// does a row past `total` or outside the out_rows of the outputs, which is not written.
US_API int us_quant_gather(const void* kc, const void* vc, const void* ks, const void* vs, const int* table,
                           int max_pages, const int* cu, const int* out_cu, int B, int total, int pages, int page,
                           int heads, int dim, int bits, void* ko, void* vo, long long ldo, int out_rows, void* stream_) {
  US_REQUIRE(B >= 0 && total >= 0 && pages >= 1 && page >= 1 && heads >= 1 && dim >= 64 && dim % 64 == 0 &&
             (bits == 8 || bits == 4) && max_pages >= 0);
  if (B == 0 || total == 0) return US_OK;
  US_REQUIRE(kc && vc && ks && vs && table && cu && ko && vo && (ldo % 8) == 0);
  US_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(ko) && aligned16(vo));
  const ReadArgs a{(const uint8_t*)kc, (const uint8_t*)vc, (const __nv_bfloat16*)ks, (const __nv_bfloat16*)vs, table, cu,
                   out_cu, (__nv_bfloat16*)ko, (__nv_bfloat16*)vo, ldo, B, max_pages, pages, page, heads, dim, total, out_rows,
                   us_status_ptr()};
  // 64 rows a block share one wait for their places; few rows are spread over more blocks
  const bool many = total >= 16384;
  auto kernel = bits == 8 ? (many ? quant_gather_kernel<8, 64> : quant_gather_kernel<8, 16>)
                          : (many ? quant_gather_kernel<4, 64> : quant_gather_kernel<4, 16>);
  const int rows = many ? 64 : 16;
  US_CUDA_CHECK(us::launch_pdl(kernel, dim3((total + rows - 1) / rows), dim3(256), 0, (cudaStream_t)stream_, a));
  return US_OK;
}

// The first min(shared[g], max_len) cached rows behind row cu_rows[g]'s page list as FP16 under the powers of two
// `exps`, to ko / vo [groups][max_len][heads][dim], and q [batch, Hq, dim] as FP16 rows qo under the factors q_back.
US_API int us_quant_prefix(const void* kc, const void* vc, const void* ks, const void* vs, const int* table, int max_pages,
                           const int* cu_rows, const int* shared, int groups, int max_len, int pages, int page, int heads,
                           int dim, int bits, const void* q, long long ldq, int batch, int Hq, void* ko, void* vo, void* qo,
                           float* q_back, void* exps, void* stream_) {
  US_REQUIRE(kc && vc && ks && vs && table && cu_rows && shared && q && ko && vo && qo && q_back && exps);
  US_REQUIRE(groups >= 1 && groups <= 65535 && max_len >= 1 && pages >= 1 && page >= 1 && heads >= 1 && dim >= 64 && dim % 64 == 0 &&
             (bits == 8 || bits == 4) && batch >= 1 && Hq >= 1 && max_pages >= 1);
  US_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(ko) && aligned16(vo));
  const PrefixArgs a{(const uint8_t*)kc, (const uint8_t*)vc, (const __nv_bfloat16*)ks, (const __nv_bfloat16*)vs, table, cu_rows,
                     shared, (const __nv_bfloat16*)q, ldq, (__half*)ko, (__half*)vo, (__half*)qo, q_back, (int2*)exps, groups,
                     max_len, max_pages, pages, page, heads, dim, batch, Hq, us_status_ptr()};
  cudaStream_t stream = (cudaStream_t)stream_;
  US_CUDA_CHECK(us::launch_pdl(prefix_scales_kernel, dim3(groups * heads + (batch * Hq + 15) / 16), dim3(512), 0, stream, a));
  US_CUDA_CHECK(us::launch_pdl(bits == 8 ? prefix_expand_kernel<8> : prefix_expand_kernel<4>,
                               dim3((max_len + kReadRows - 1) / kReadRows, groups, 2), dim3(256), 0, stream, a));
  return US_OK;
}
