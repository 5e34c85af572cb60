// Softmax attention of one new token a sequence over cache pages: scores capped by a tanh, biased by distance, cut
// below a first visible key or a window; pages of bf16, or of 8- or 4-bit integers (quant_pages.cu); batches whose
// sequences share a prefix, whose part of the result comes from scored_flash_tc05.cu.
//
//   s = scale q.k_j;  s = cap tanh(s / cap);  s -= slope_h (p - j), p = length - 1;  first <= j < length
//   out_h = sum_j e^s v_j / sum_j e^s                       (zeros where no key is visible)
//
// Bound by the bytes of the keys, so everything serves the stream of loads:
//
// * All keys of the launch form one list of tiles ordered by (sequence, key head, tile), cut into one range per warp: no
//   SM idles behind a long sequence, and no warp waits for another before its range is done.  A warp fills its own
//   ring of stages (the K rows or the V rows of a tile) with 16-byte asynchronous copies, on across pairs; page ids of
//   a tile are one load per lane, a tile ahead of its copies.
// * A pair (sequence, key head) inside one range is written by its warp.  Others leave unnormalised outputs, maxima and
//   sums: of the pair that a range ends in, in the warp's ring, which is free by then; of one that it only begins in, in the
//   warp's slot in memory.  At the end all warps of a CTA fold the parts of its pairs, sixteen channels of a pair at a
//   time, and pairs that go on in other CTAs once more through the CTAs' slots, by the CTA whose arrival completes a
//   pair's count and puts it back to zero.  (Warps that split every tile between them and met at each pair's end spent a
//   quarter of the time there.)  Both rounds are one short loop: every instruction of this end is fetched cold, by all
//   SMs at once, and an unrolled form of it took 15 us where this one takes some 8.
// * Keys stand on the M side of m16n8k16 products (S^T = K Q^T, O^T = V^T P^T), the query heads of a key head on the
//   N side: groups of up to 8 heads pay for 8 columns, not for 16 rows, and the softmax has its maximum and sum
//   per column, three shuffles each.  P^T becomes the B operand by an 8 x 8 transpose in registers (movmatrix).
// * Integer codes are multiplied as FP16 numbers 1024 + u or 64 + u, u the code plus 128 or 8, which bit operations form
//   (a byte in the last bits of 1024, a nibble four bits up in those of 64).  The offset is taken out by products as
//   well: -offset x Q starts the sums of K, ones x P^T gives the sums that V's outputs have too much, tile by tile.
//   One and a half (8 bits) or one and three quarters (4 bits) instructions two codes.  (Nibbles in the last bits of
//   1024 take half an instruction less, but an offset of 344 times their size eats as much of FP32's sums.)  Scales
//   never touch the codes: a key's
//   multiply its scores, a value's its probabilities.  Which channel stands in which k slot is free as long as Q
//   agrees, so bytes and nibbles are taken out of the words as they lie; for V the free order is that of the output.
//
// Statistics and outputs are FP32.  P is rounded once for its product: to bf16 (2^-8 of a weight at most), or, over
// integer pages, with its value's scale to FP16 (2^-11).  There the weights are held as p s 2^(14 - E), E the exponent
// of the largest value scale so far: 15 bits above 1 and 24 below, so a value 2^10 times its neighbours' costs them
// nothing.  Q is divided by the power of two of its largest channel to be FP16 exactly (channels under 2^-14 of that lose
// bits).  Keys that are not visible are never loaded (zeros in their place): nothing in them reaches the result.
//
// 64 sequences of up to 7,000 keys, 32 / 4 heads of 128: bf16 98 us (the loads alone take 94), 8 bits 64 us, 4 bits 57 us;
// there instructions bound it, and the 8 us of the end.
#include <type_traits>
#include "include/us_common.cuh"
#include "include/us_mma.cuh"

namespace {

constexpr int kMaxSeqs = 704;               // of a launch: what the ring leaves of shared memory

struct DecodeArgs {
  const __nv_bfloat16* q;
  const uint8_t *kc, *vc;
  const __nv_bfloat16 *ks, *vs;             // scales of integer pages
  const int *table, *lens, *starts;
  __nv_bfloat16* out;
  // parts: of warps, one each, then of CTAs, two each (kPart floats a part, see there)
  float* part;
  int* counters;                            // [B * pairs per sequence], zero between launches
  const float* slopes;
  long long ldq, ldo;
  int B, Hq, Hkv, chunks, max_pages, pages, page, shift, window;
  float scale_log2, scale_cap, cap_log2;    // cap_log2 == 0: no cap; scale_cap = 2 scale log2(e) / cap
  // shared prefixes: rows [cu_rows[g], cu_rows[g + 1]) share their first min(shared[g], most_shared) keys, which are not this
  // launch's; its results then go unnormalised to own_o [B][Hq][D], own_ml [B][Hq][2] for scored_merge_kernel
  const int *cu_rows, *shared;
  float *own_o, *own_ml;
  int groups, most_shared, most_rows;       // most_rows: of a group
  unsigned int* status;
  uint32_t magic;                           // see bytes_even, nibbles
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // 8 x 8 matrix of 16-bit values across the warp
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp16z(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4z(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8] in bf16 or FP16.  Not volatile: products of unlike sums may pass one another.
__device__ __forceinline__ void mma_b(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_h(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Bytes 0 and 2, or 1 and 3, of a word of codes plus 128 as 1024 + u; nibbles 0 and 4 of a word of codes plus 8 as 64 + u,
// for the others the word is shifted.  `magic` (0x64646464, 0x54005400) comes as a kernel argument: as a constant it was
// moved into a register anew before most of its uses, a third of all instructions.
__device__ __forceinline__ uint32_t bytes_even(uint32_t x, uint32_t magic) { return __byte_perm(x, magic, 0x4240); }
__device__ __forceinline__ uint32_t bytes_odd(uint32_t x, uint32_t magic) { return __byte_perm(x, magic, 0x4341); }
__device__ __forceinline__ uint32_t nibbles(uint32_t x, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(y) : "r"(x), "r"(magic));     // (x & mask) | magic
  return y;
}
constexpr uint32_t kOne = 0x3C003C00u;          // FP16 pairs: 1, -1152 = -(1024 + 128), -72 = -(64 + 8)
constexpr uint32_t kMinus1152 = 0xE480E480u, kMinus72 = 0xD480D480u;
__device__ __forceinline__ float power_of_two(int field) {     // 2^(field - 127), field clamped to what a float has
  return __uint_as_float((uint32_t)min(max(field, 0), 254) << 23);
}

// The group with whose rows row b shares keys, or -1.  A group that begins before the batch has no page list to read, and rows
// past those that the prefix launch was planned for are not in its results: such rows have all their keys to themselves, and the
// status says so.
__device__ __forceinline__ int group_of(const int* cu_rows, int groups, int b, int most_rows, unsigned int* status) {
  int g = 0, h = groups - 1;
  while (g < h) {
    const int mid = (g + h + 1) >> 1;
    if (cu_rows[mid] <= b) g = mid; else h = mid - 1;
  }
  const int first = cu_rows[g], end = cu_rows[g + 1];
  if (b < first || b >= end) return -1;
  if (first >= 0 && b - first < most_rows) return g;
  us_dev_fail(status, US_DEV_BOUNDS);
  return -1;
}

// A position in the tile list.
struct Walk {
  int b, hc, t, tiles;
};

template <int D, int FMT, int NT>           // FMT: bits of a code (16: bf16)
struct Shape {
  // Integer codes take more instructions a byte, and with two warps a scheduler each waits for itself: sixteen warps of
  // 128 registers, or, where a byte holds two codes, twelve of 168 with 64 keys each (32 sequences of about 8,000 keys, 8
  // key heads of 128 channels, 4 bits: 57 us, sixteen of 32 keys 63).  Two head tiles want the registers of eight warps:
  // twelve spill, 137 us in place of 86.
  static constexpr int kWarps = FMT == 16 || NT == 2 ? 8 : FMT == 8 ? 16 : 12;
  static constexpr int kRow = D * FMT / 8;                          // bytes of a cached row
  static constexpr int kKeys = NT == 1 && (FMT == 16 ? kRow <= 128 : FMT == 4) ? 64 : 32;   // keys of a warp's part of a tile
  static constexpr int kScales = FMT == 16 ? 0 : kKeys * 4;
  static constexpr int kStage = kKeys * kRow + kScales;             // K or V rows of it
  static constexpr int kRoom = (FMT == 16 ? 196608 : 202752) / kWarps;    // ring bytes of a warp
  static constexpr int kStages = kRoom / kStage > 8 ? 8 : kRoom / kStage;
  static constexpr int kPieces = kRow / 16;                         // 16-byte pieces of a row
  static_assert(kStages >= 3, "ring");
};

template <int PIECES>
__device__ __forceinline__ int swizzle(int row, int piece) {        // eight rows' same piece: eight bank groups
  if constexpr (PIECES >= 8) return piece ^ (row & 7);
  else if constexpr (PIECES == 4) return piece ^ ((row >> 1) & 3);
  else return piece ^ ((row >> 2) & 1);
}

// A part of a pair's result (see kPart): where it is, and which pair's, by its first tile.
struct Part {
  const float* at;                          // null: none
  int begin, end, b, hc;
};

template <int D, int FMT, int NT>
constexpr size_t shared_bytes() {
  using S = Shape<D, FMT, NT>;
  return (size_t)S::kWarps * S::kRoom + 32 * sizeof(Part) + 16 + (3 * kMaxSeqs + 4) * 4;   // rings; parts; flags; sequences
}

template <int D, int FMT, int NT>           // NT: 8-column head tiles (query heads of a key head in one pass: 8 NT)
__global__ void __launch_bounds__((Shape<D, FMT, NT>::kWarps * 32), 1) scored_decode_kernel(const DecodeArgs a) {
  using S = Shape<D, FMT, NT>;
  constexpr int kWarps = S::kWarps, kThreads = kWarps * 32;
  constexpr int KW = S::kKeys, MT = KW / 16, KS = D / 16, G = D / 64, KL = KW / 32;
  // beside the launch of the shared prefixes, which waited for what both read before it let this one start
  if (a.groups > 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  else US_PDL_PROLOGUE();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem + (size_t)warp * S::kRoom;
  Part* parts = (Part*)(smem + (size_t)kWarps * S::kRoom);  // [warp][2]: begun before its range, ended by it
  int* flag = (int*)(parts + 32);           // [2] CTAs of its first, last pair if this CTA completes it (else 0), [2] first of them
  int* pre = flag + 4;                      // tiles before sequence b
  int* first = pre + kMaxSeqs + 4;          // visible keys of sequence b: [first, end)
  int* end = first + kMaxSeqs;

  // ---- the tile list ----
  const int B = a.B, Hc = a.Hkv * a.chunks;
  for (int b = tid; b < B; b += kThreads) {
    int len = max(a.lens[b], 0), lo = a.starts ? max(a.starts[b], 0) : 0;
    if (a.window > 0) lo = max(lo, len - a.window);
    if (a.groups > 0) {
      const int g = group_of(a.cu_rows, a.groups, b, a.most_rows, a.status);
      if (g >= 0) lo = max(lo, min(a.shared[g], a.most_shared));
    }
    const long long room = (long long)a.max_pages * a.page;
    int hi = len;
    if (hi > room) {
      hi = (int)room;
      us_dev_fail(a.status, US_DEV_BOUNDS);
    }
    lo = min(lo, hi);
    first[b] = lo;
    end[b] = hi;
    pre[b + 1] = max(1, (hi - lo + KW - 1) / KW);       // a pair without keys still has its zeros to write
  }
  if (tid == 0) pre[0] = 0;
  __syncthreads();
  if (warp == 0) {
    const int per = (B + 31) / 32;
    const int l0 = 1 + lane * per, l1 = min(B + 1, l0 + per);
    int s = 0;
    for (int i = l0; i < l1; ++i) s += pre[i];
    int ps = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, ps, o);
      if (lane >= o) ps += v;
    }
    int run = ps - s;
    for (int i = l0; i < l1; ++i) {
      run += pre[i];
      pre[i] = run;
    }
  }
  __syncthreads();
  const int total = Hc * pre[B];
  // One range of the list a warp.  Where there are fewer tiles than warps, every CTA has as many warps at work, and as
  // many that a pair of average length ends in eight CTAs' parts at most: 32 of one warp each cost a request of 1021 keys
  // 4 us at the end.
  const int ctas = gridDim.x, cta = blockIdx.x;
  const int active = min(kWarps, max((total + ctas - 1) / ctas, (pre[B] + 8 * B - 1) / (8 * B))), workers = min(total, ctas * active);
  const unsigned long long pace = ((unsigned long long)total << 32) / (unsigned)workers;
  auto start_of = [&](int k) -> int { return k >= workers ? total : (int)((pace * (unsigned)k) >> 32); };
  auto worker_of = [&](int g) -> int {
    int k = min((int)((float)g * ((float)workers / (float)total)), workers - 1);
    while (k + 1 < workers && start_of(k + 1) <= g) ++k;
    while (k > 0 && start_of(k) > g) --k;
    return k;
  };
  const int me0 = cta * active, me1 = min(me0 + active, workers), me = me0 + warp;     // this CTA's ranges, this warp's
  if (me0 >= workers) return;
  const bool works = warp < active && me < workers;
  const int g0 = works ? start_of(me) : total, g1 = works ? start_of(me + 1) : total;
  // the pair that tile g is in
  auto find = [&](int g) -> Walk {
    Walk w;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (Hc * pre[mid] <= g) lo = mid; else hi = mid - 1;
    }
    w.b = lo;
    w.tiles = pre[lo + 1] - pre[lo];
    const int r = g - Hc * pre[lo];
    w.hc = r / w.tiles;
    w.t = r - w.hc * w.tiles;
    return w;
  };
  Walk load = find(min(g0, total - 1));
  Walk cur = load;
  auto advance = [&](Walk& w) {
    if (++w.t < w.tiles) return;
    w.t = 0;
    if (++w.hc < Hc) return;
    w.hc = 0;
    ++w.b;
    if (w.b < B) w.tiles = pre[w.b + 1] - pre[w.b];
  };

  // ---- loads: this warp's keys of a tile, K rows into one stage, V rows into the next ----
  // Place of a key in the cache in units of 16 bytes; kNone where there is nothing to load.
  constexpr uint32_t kNone = 0xffffffffu;
  const uint32_t per_slot = (uint32_t)a.Hkv * S::kPieces;
  auto place_of = [&](const Walk& w, uint32_t (&at)[KL], uint32_t (&spot)[KL]) {    // of key head 0; spot: of its scales
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int j = first[w.b] + w.t * KW + i * 32 + lane;
      at[i] = kNone;
      spot[i] = 0;
      if (j < end[w.b]) {
        const int pi = a.shift >= 0 ? j >> a.shift : j / a.page;
        const int pg = __ldg(a.table + (long long)w.b * a.max_pages + pi);
        if ((unsigned)pg < (unsigned)a.pages) {
          const uint32_t base = (uint32_t)(pg * a.page), off = (uint32_t)(j - pi * a.page);
          at[i] = (base + off) * per_slot;
          if constexpr (FMT != 16) spot[i] = base * (uint32_t)a.Hkv + off;
        } else {
          us_dev_fail(a.status, US_DEV_BOUNDS);
        }
      }
    }
  };
  int loaded = g0;                          // tiles whose K rows have been asked for
  uint32_t next_place[KL], next_spot[KL], place[KL], spot[KL];
  bool full_now = false, more = true;
  if (works) place_of(load, next_place, next_spot);
  // the next stage's copies: V_ROWS: of the tile whose K rows went last; else of the next tile
  auto issue = [&](auto v_rows, uint32_t to) {
    constexpr bool kV = decltype(v_rows)::value;
    if constexpr (!kV) {
      more = loaded < g1;
      if (more) {
        const uint32_t hk = (uint32_t)(a.chunks == 1 ? load.hc : load.hc / a.chunks);
        bool full = true;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const bool there = next_place[i] != kNone;
          full &= there;
          place[i] = there ? next_place[i] + hk * S::kPieces : kNone;
          if constexpr (FMT != 16) spot[i] = next_spot[i] + hk * (uint32_t)a.page;
        }
        full_now = __all_sync(0xffffffffu, full);
        ++loaded;
        if (loaded < g1) {
          advance(load);
          place_of(load, next_place, next_spot);
        }
      }
    }
    if (more) {
      constexpr int kRows = 32 / S::kPieces;       // rows that one instruction of the warp brings
      const int piece = lane % S::kPieces, r0 = lane / S::kPieces;
      const uint8_t* base = (kV ? a.vc : a.kc) + piece * 16;
      if (full_now) {
#pragma unroll
        for (int i = 0; i < KW / kRows; ++i) {
          const int r = i * kRows + r0;
          const uint32_t at = __shfl_sync(0xffffffffu, place[i * kRows / 32], r & 31);
          us::cp16(to + r * S::kRow + swizzle<S::kPieces>(r, piece) * 16, base + (unsigned long long)at * 16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW / kRows; ++i) {
          const int r = i * kRows + r0;
          const uint32_t at = __shfl_sync(0xffffffffu, place[i * kRows / 32], r & 31);
          cp16z(to + r * S::kRow + swizzle<S::kPieces>(r, piece) * 16, base + (at == kNone ? 0ull : (unsigned long long)at * 16), at != kNone);
        }
      }
      if constexpr (FMT != 16) {            // 4 bytes of scales a key: two groups, or one beside its neighbour's
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const bool there = place[i] != kNone;
          const uint32_t word = there ? (G == 2 ? spot[i] : spot[i] >> 1) : 0;
          cp4z(to + KW * S::kRow + (i * 32 + lane) * 4, (const uint8_t*)(kV ? a.vs : a.ks) + (unsigned long long)word * 4, there);
        }
      }
    }
    us::cp_commit();
  };

  const int c4 = lane & 3, r8 = lane >> 2;
  const uint32_t magic = a.magic;
  // where this lane's rows of the 8 x 8 matrices of a piece are in a stage (bf16: K's and V's differ in their order)
  constexpr int kLoads = FMT == 16 ? KS : S::kPieces / 2;
  uint32_t k_lane[kLoads], v_lane[FMT == 16 ? KS : 1];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    k_lane[i] = (lane & 15) * S::kRow + swizzle<S::kPieces>(lane & 15, 2 * i + (lane >> 4)) * 16;
    if constexpr (FMT == 16) {
      const int row = (lane & 7) + (lane >> 4) * 8;
      v_lane[i] = row * S::kRow + swizzle<S::kPieces>(row, 2 * i + ((lane >> 3) & 1)) * 16;
    }
  }
  uint32_t qf[NT][KS][2];
  float m[NT][2], l[NT][2], bias[NT][2], factor[NT][2], o[KS][NT][4], offset[G][NT][2];
  int top_scale = 0;                         // exponent field of the largest value scale so far (integer pages)
  auto begin_pair = [&]() {
    const int share = a.Hq / a.Hkv, hk = a.chunks == 1 ? cur.hc : cur.hc / a.chunks, chunk = cur.hc - hk * a.chunks;
    top_scale = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int gi = chunk * 16 + nt * 8 + r8;
      const __nv_bfloat16* row = a.q + (long long)cur.b * a.ldq + (long long)(hk * share + gi) * D;
      const bool there = gi < share;
      float back = 1.f;                      // what the head's scores are multiplied by
#pragma unroll
      for (int k = 0; k < KS; ++k) qf[nt][k][0] = qf[nt][k][1] = 0;
      if constexpr (FMT == 16) {
        if (there) {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            qf[nt][k][0] = *reinterpret_cast<const uint32_t*>(row + k * 16 + c4 * 2);
            qf[nt][k][1] = *reinterpret_cast<const uint32_t*>(row + k * 16 + c4 * 2 + 8);
          }
        }
      } else {
        // bf16 pairs of the slots, then FP16 under the power of two of the head's largest channel
        if (there) {
          if constexpr (FMT == 8) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              const uint2 w = *reinterpret_cast<const uint2*>(row + k * 16 + c4 * 4);
              qf[nt][k][0] = __byte_perm(w.x, w.y, 0x5410);
              qf[nt][k][1] = __byte_perm(w.x, w.y, 0x7632);
            }
          } else {
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
              const uint4 w = *reinterpret_cast<const uint4*>(row + k * 16 + c4 * 8);
              qf[nt][k][0] = __byte_perm(w.x, w.z, 0x5410);
              qf[nt][k][1] = __byte_perm(w.x, w.z, 0x7632);
              qf[nt][k + 1][0] = __byte_perm(w.y, w.w, 0x5410);
              qf[nt][k + 1][1] = __byte_perm(w.y, w.w, 0x7632);
            }
          }
        }
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k) most = __vmaxu2(most, __vmaxu2(qf[nt][k][0] & 0x7fff7fffu, qf[nt][k][1] & 0x7fff7fffu));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // (the ends of the range beside the ones that have a reciprocal: channels of up to 4, and under 1)
        const int e = min(max((int)(max(most & 0xffffu, most >> 16) >> 7), 1), 253);
        const float down = power_of_two(254 - e);
        back = power_of_two(e);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = qf[nt][k][i];
            qf[nt][k][i] = pack_h(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
          }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          constexpr uint32_t kOff = FMT == 8 ? kMinus1152 : kMinus72;
#pragma unroll
          for (int k = 4 * g; k < 4 * g + 4; ++k) mma_h(acc, kOff, kOff, kOff, kOff, qf[nt][k][0], qf[nt][k][1]);
          offset[g][nt][0] = acc[0];
          offset[g][nt][1] = acc[1];
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = chunk * 16 + nt * 8 + c4 * 2 + e;
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
        bias[nt][e] = a.slopes && h < share ? a.slopes[hk * share + h] * 1.4426950408889634f : 0.f;
        factor[nt][e] = (a.cap_log2 > 0.f ? a.scale_cap : a.scale_log2) * (FMT == 16 ? 1.f : __shfl_sync(0xffffffffu, back, (c4 * 2 + e) * 4));
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
    }
    float least = fminf(bias[0][0], bias[0][1]);
    if constexpr (NT == 2) least = fminf(least, fminf(bias[1][0], bias[1][1]));
    if (least < 0.f) us_dev_fail(a.status, US_DEV_BOUNDS);
  };

  // a key's scales out of a stage: two, or (64 channels) the one whose half its parity says, the page size being even
  auto scales = [&](const uint32_t* st, int key, int j0, float (&f)[G]) {
    const uint32_t w = st[key];
    if constexpr (G == 2) {
      f[0] = __uint_as_float(w << 16);
      f[1] = __uint_as_float(w & 0xffff0000u);
    } else {
      f[0] = __uint_as_float((j0 + key) & 1 ? w & 0xffff0000u : w << 16);
    }
  };

  float s[MT][NT][4];                        // scores of a tile, then its weights
  float alpha[NT][2];                        // what the outputs so far are multiplied by
  bool grown = false;
  // ---- K rows of a stage: S^T = K Q^T and the softmax's step ----
  auto consume_k = [&](const uint8_t* st) {
    const int j0 = first[cur.b] + cur.t * KW, hi = end[cur.b];
    if (j0 >= hi) return;
    const uint32_t kd = (uint32_t)__cvta_generic_to_shared(st);
    const uint32_t* sk = reinterpret_cast<const uint32_t*>(st + KW * S::kRow);
    // a piece of channels at a time over all keys: MT sums that do not wait for one another
    if constexpr (FMT == 16) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint32_t from = kd + k_lane[k];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t f[4];
          us::ldsm4(f, from + mt * 16 * S::kRow);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_b(s[mt][nt], f[0], f[1], f[2], f[3], qf[nt][k][0], qf[nt][k][1]);
        }
      }
    } else {
      float acc[MT][G][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[mt][g][nt][e] = offset[g][nt][e & 1];
#pragma unroll
      for (int i = 0; i < S::kPieces / 2; ++i) {
        const uint32_t from = kd + k_lane[i];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t f[4];
          us::ldsm4(f, from + mt * 16 * S::kRow);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t x = f[2 * half], y = f[2 * half + 1];   // keys 0 - 7 and 8 - 15
            const int piece = 2 * i + half;
            if constexpr (FMT == 8) {
              x ^= 0x80808080u;
              y ^= 0x80808080u;
              const uint32_t a0 = bytes_even(x, magic), a1 = bytes_even(y, magic), a2 = bytes_odd(x, magic), a3 = bytes_odd(y, magic);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_h(acc[mt][piece / 4][nt], a0, a1, a2, a3, qf[nt][piece][0], qf[nt][piece][1]);
            } else {
              const uint32_t a0 = nibbles(x << 4, magic), a1 = nibbles(y << 4, magic), a2 = nibbles(x, magic), a3 = nibbles(y, magic);
              const uint32_t b0 = nibbles(x >> 4, magic), b1 = nibbles(y >> 4, magic), b2 = nibbles(x >> 8, magic), b3 = nibbles(y >> 8, magic);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_h(acc[mt][piece / 2][nt], a0, a1, a2, a3, qf[nt][2 * piece][0], qf[nt][2 * piece][1]);
                mma_h(acc[mt][piece / 2][nt], b0, b1, b2, b3, qf[nt][2 * piece + 1][0], qf[nt][2 * piece + 1][1]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float f0[G], f1[G];
        scales(sk, mt * 16 + r8, j0, f0);
        scales(sk, mt * 16 + r8 + 8, j0, f1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = acc[mt][0][nt][e] * (e < 2 ? f0[0] : f1[0]);
            if constexpr (G == 2) x = fmaf(acc[mt][1][nt][e], e < 2 ? f0[1] : f1[1], x);
            s[mt][nt][e] = x;
          }
      }
    }
    // scores in units of log2(e)
    if (a.cap_log2 > 0.f) {                  // tanh y = 1 - 2 / (1 + e^(2 y)): off by some 2^-22 of the cap
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[mt][nt][e] = fmaf(-2.f * a.cap_log2, rcp(1.f + ex2(s[mt][nt][e] * factor[nt][e & 1])), a.cap_log2);
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] *= factor[nt][e & 1];
    }
    if (a.slopes) {
      const int away0 = a.lens[cur.b] - 1 - j0 - r8;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float away = (float)(away0 - mt * 16 - h * 8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[mt][nt][2 * h + e] = fmaf(-bias[nt][e], away, s[mt][nt][2 * h + e]);
        }
    }
    if (j0 + KW > hi) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j0 + mt * 16 + r8 + (e >> 1) * 8 >= hi) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[mt][nt][e] = -INFINITY;
          }
    }
    grown = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
        for (int mt = 1; mt < MT; ++mt) t = fmaxf(t, fmaxf(s[mt][nt][e], s[mt][nt][e + 2]));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        t = fmaxf(t, m[nt][e]);
        alpha[nt][e] = t == -INFINITY ? 1.f : ex2(m[nt][e] - t);
        grown |= t > m[nt][e];
        m[nt][e] = t;
        const float base = t == -INFINITY ? 0.f : t;      // no score above -inf so far: weights of zero
        float sum = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p = ex2(s[mt][nt][e + 2 * h] - base);
            s[mt][nt][e + 2 * h] = p;
            sum += p;
          }
        l[nt][e] = fmaf(l[nt][e], alpha[nt][e], sum);
      }
    grown = __any_sync(0xffffffffu, grown);
  };
  // ---- V rows of a stage: O^T += V^T P^T ----
  auto consume_v = [&](const uint8_t* st) {
    const int j0 = first[cur.b] + cur.t * KW;
    if (j0 >= end[cur.b]) return;
    const uint32_t vd = (uint32_t)__cvta_generic_to_shared(st);
    const uint32_t* sv = reinterpret_cast<const uint32_t*>(st + KW * S::kRow);
    float lift = 1.f;                        // 2^(14 - E)
    float shrink = 1.f;
    if constexpr (FMT != 16) {
      // Scales are not negative: as integers they are in order.  One that is no number has no part in this: its group's outputs
      // are lost, those of the other group are not.
      uint32_t big = 0;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        float f[G];
        scales(sv, i * 32 + lane, j0, f);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t x = __float_as_uint(f[g]) & 0x7fffffffu;
          big = max(big, x < 0x7f800000u ? x : 0u);
        }
      }
      const int e = max(top_scale, (int)(__reduce_max_sync(0xffffffffu, big) >> 23));
      shrink = power_of_two(127 - (e - top_scale));
      top_scale = e;
      lift = power_of_two(268 - e);
    }
    // the weights as the second operand of the products
    constexpr int GP = FMT == 16 ? 1 : G;
    uint32_t pb[MT][GP][NT][2];
    if constexpr (FMT == 16) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pb[mt][0][nt][0] = transposed(us::pack_bf(s[mt][nt][0], s[mt][nt][1]));
          pb[mt][0][nt][1] = transposed(us::pack_bf(s[mt][nt][2], s[mt][nt][3]));
        }
      if (grown) {
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] *= alpha[nt][e & 1];
      }
    } else {
      float sums[G][NT][4];                  // of the rounded weights
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sums[g][nt][e] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float f0[G], f1[G];
        scales(sv, mt * 16 + r8, j0, f0);
        scales(sv, mt * 16 + r8 + 8, j0, f1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          f0[g] *= lift;
          f1[g] *= lift;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            pb[mt][g][nt][0] = transposed(pack_h(s[mt][nt][0] * f0[g], s[mt][nt][1] * f0[g]));
            pb[mt][g][nt][1] = transposed(pack_h(s[mt][nt][2] * f1[g], s[mt][nt][3] * f1[g]));
            mma_h(sums[g][nt], kOne, kOne, kOne, kOne, pb[mt][g][nt][0], pb[mt][g][nt][1]);
          }
        }
      }
      // the outputs so far under the new maximum, and less what this tile's offsets will add
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = alpha[nt][e] * shrink;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const float less = sums[g][nt][e] * (FMT == 4 ? -72.f : -1152.f);
#pragma unroll
            for (int i = 4 * g; i < 4 * g + 4; ++i) {
              o[i][nt][e] = fmaf(o[i][nt][e], f, less);
              o[i][nt][e + 2] = fmaf(o[i][nt][e + 2], f, less);
            }
          }
        }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t f[4];
        if constexpr (FMT == 16) {
          us::ldsm4t(f, vd + v_lane[i] + mt * 16 * S::kRow);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_b(o[i][nt], f[0], f[1], f[2], f[3], pb[mt][0][nt][0], pb[mt][0][nt][1]);
        } else {
          us::ldsm4t(f, vd + k_lane[i] + mt * 16 * S::kRow);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t x = f[2 * half], y = f[2 * half + 1];   // keys 0 - 7 and 8 - 15
            const int piece = 2 * i + half;
            if constexpr (FMT == 8) {
              x ^= 0x80808080u;
              y ^= 0x80808080u;
              const uint32_t a0 = bytes_even(x, magic), a1 = bytes_odd(x, magic), a2 = bytes_even(y, magic), a3 = bytes_odd(y, magic);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_h(o[piece][nt], a0, a1, a2, a3, pb[mt][piece / 4][nt][0], pb[mt][piece / 4][nt][1]);
            } else {
              const uint32_t a0 = nibbles(x << 4, magic), a1 = nibbles(x, magic), a2 = nibbles(y << 4, magic), a3 = nibbles(y, magic);
              const uint32_t b0 = nibbles(x >> 4, magic), b1 = nibbles(x >> 8, magic), b2 = nibbles(y >> 4, magic), b3 = nibbles(y >> 8, magic);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_h(o[2 * piece][nt], a0, a1, a2, a3, pb[mt][piece / 2][nt][0], pb[mt][piece / 2][nt][1]);
                mma_h(o[2 * piece + 1][nt], b0, b1, b2, b3, pb[mt][piece / 2][nt][0], pb[mt][piece / 2][nt][1]);
              }
            }
          }
        }
      }
    }
  };
  // channel of output row i of accumulator tile t
  auto channel = [&](int t, int half) {
    if constexpr (FMT == 16) return t * 16 + r8 + half * 8;
    else if constexpr (FMT == 8) return t * 16 + r8 * 2 + half;
    else return (t >> 1) * 32 + r8 * 4 + (t & 1) * 2 + half;
  };

  // writes N accumulator tiles from t0 on (unnormalised, under maximum M with sum L)
  auto finish = [&](auto tiles, int t0, float (*acc)[NT][4], int b, int hc, const float (&M)[NT][2], const float (&L)[NT][2]) {
    constexpr int N = decltype(tiles)::value;
    const int share = a.Hq / a.Hkv, hk = a.chunks == 1 ? hc : hc / a.chunks, chunk = hc - hk * a.chunks;
    const int heads = min(8 * NT, share - chunk * 16);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = nt * 8 + c4 * 2 + e;
        if (h >= heads) continue;
        const int head = hk * share + chunk * 16 + h;
        if (a.groups > 0) {
          const long long row = (long long)b * a.Hq + head;
#pragma unroll
          for (int t = 0; t < N; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) a.own_o[row * D + channel(t0 + t, half)] = acc[t][nt][e + 2 * half];
          if (t0 == 0 && r8 == 0) *reinterpret_cast<float2*>(a.own_ml + row * 2) = make_float2(M[nt][e], L[nt][e]);
          continue;
        }
        const float inv = L[nt][e] == 0.f ? 0.f : 1.f / L[nt][e];
        __nv_bfloat16* to = a.out + (long long)b * a.ldo + (long long)head * D;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int half = 0; half < 2; ++half) to[channel(t0 + t, half)] = us::f2bf(acc[t][nt][e + 2 * half] * inv);
      }
  };
  // A part: outputs in the order of the accumulators [NT][D / 16][32 lanes][4], then maxima and sums [NT * 8][2].
  constexpr int kPart = NT * (KS * 128 + 16);
  static_assert(2 * kPart * 4 <= S::kRoom, "two parts have room in a ring");
  auto store_tile = [&](float* part, int t, const float (&x)[NT][4]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      *reinterpret_cast<float4*>(part + ((nt * KS + t) * 32 + lane) * 4) = make_float4(x[nt][0], x[nt][1], x[nt][2], x[nt][3]);
  };
  auto store_sums = [&](float* part, const float (&M)[NT][2], const float (&L)[NT][2]) {
    if (r8 == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        *reinterpret_cast<float4*>(part + NT * KS * 128 + (nt * 8 + c4 * 2) * 2) = make_float4(M[nt][0], L[nt][0], M[nt][1], L[nt][1]);
    }
  };
  auto ring_of = [&](int w) { return (float*)(smem + (size_t)w * S::kRoom); };
  // a value under maximum x into one under M
  auto join = [&](float x, float& M, float& f, float& w) {
    const float top = fmaxf(M, x);
    f = M == -INFINITY ? 0.f : ex2(M - top);
    w = ex2(x - top);
    M = top;
  };
  // accumulator tile t of up to four parts into acc under maxima M with sums L.  A maximum of -inf: no key has a weight and the
  // sum is zero, or no score is a number and the sum is none, which then is the pair's sum too (its outputs may hold anything).
  auto add_parts = [&](const float* (&at)[4], int t, float (&acc)[1][NT][4], float (&M)[NT][2], float (&L)[NT][2]) {
    float4 v[4][NT], p[4][NT];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        v[k][nt] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
        if (at[k]) {
          v[k][nt] = *reinterpret_cast<const float4*>(at[k] + NT * KS * 128 + nt * 16 + c4 * 4);
          p[k][nt] = *reinterpret_cast<const float4*>(at[k] + ((nt * KS + t) * 32 + lane) * 4);
        }
      }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f, w;
        if (v[k][nt].x == -INFINITY) {
          L[nt][0] += v[k][nt].y;
        } else {
          join(v[k][nt].x, M[nt][0], f, w);
          L[nt][0] = fmaf(w, v[k][nt].y, L[nt][0] * f);
          acc[0][nt][0] = fmaf(w, p[k][nt].x, acc[0][nt][0] * f);
          acc[0][nt][2] = fmaf(w, p[k][nt].z, acc[0][nt][2] * f);
        }
        if (v[k][nt].z == -INFINITY) {
          L[nt][1] += v[k][nt].w;
        } else {
          join(v[k][nt].z, M[nt][1], f, w);
          L[nt][1] = fmaf(w, v[k][nt].w, L[nt][1] * f);
          acc[0][nt][1] = fmaf(w, p[k][nt].y, acc[0][nt][1] * f);
          acc[0][nt][3] = fmaf(w, p[k][nt].w, acc[0][nt][3] * f);
        }
      }
  };
  // a whole part
  auto add_part = [&](const float* part, float (*acc)[NT][4], float (&M)[NT][2], float (&L)[NT][2]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float4 v = *reinterpret_cast<const float4*>(part + NT * KS * 128 + nt * 16 + c4 * 4);
      float4 p[KS];
#pragma unroll
      for (int t = 0; t < KS; ++t) p[t] = *reinterpret_cast<const float4*>(part + ((nt * KS + t) * 32 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = e ? v.z : v.x;
        if (x == -INFINITY) {
          L[nt][e] += e ? v.w : v.y;
          continue;
        }
        float f, w;
        join(x, M[nt][e], f, w);
        L[nt][e] = fmaf(w, e ? v.w : v.y, L[nt][e] * f);
#pragma unroll
        for (int t = 0; t < KS; ++t) {
          acc[t][nt][e] = fmaf(w, e ? p[t].y : p[t].x, acc[t][nt][e] * f);
          acc[t][nt][e + 2] = fmaf(w, e ? p[t].w : p[t].z, acc[t][nt][e + 2] * f);
        }
      }
    }
  };

  // ---- this warp's range ----
  constexpr int NS = S::kStages;
  using KRows = std::false_type;
  using VRows = std::true_type;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  if (tid < 32) parts[tid].at = nullptr;
  __syncthreads();
  if (works) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (i & 1) issue(VRows{}, ring_at + i * S::kStage);
      else issue(KRows{}, ring_at + i * S::kStage);
    }
    int stage = 0, i = g0, done = 0;
    const int paced = total / workers, present = me1 - me0;
    auto step = [&]() { stage = stage + 1 == NS ? 0 : stage + 1; };
    while (i < g1) {
      begin_pair();
      const int n = min(cur.tiles - cur.t, g1 - i);
      const bool from_start = cur.t == 0, to_end = cur.t + n == cur.tiles;
      for (int t = 0; t < n; ++t, ++i, ++cur.t) {
        us::cp_wait<NS - 1>();
        __syncwarp();
        consume_k(ring + stage * S::kStage);
        __syncwarp();
        // the freed stage gets what comes NS stages later: K rows if NS is even, else V rows
        if constexpr (NS % 2 == 0) issue(KRows{}, ring_at + stage * S::kStage);
        else issue(VRows{}, ring_at + stage * S::kStage);
        step();
        us::cp_wait<NS - 1>();
        __syncwarp();
        consume_v(ring + stage * S::kStage);
        __syncwarp();
        if constexpr (NS % 2 == 0) issue(VRows{}, ring_at + stage * S::kStage);
        else issue(KRows{}, ring_at + stage * S::kStage);
        step();
        // bf16: in step (every range has at least `paced` tiles), or the scheduler's favourites are done a tenth earlier
        // than the rest, whose loads alone do not fill the memory (64 x 4240 keys: 105 -> 102 us).  Integer pages
        // are bound by instructions, and waiting costs them 8 us there.
        if (FMT == 16 && ++done < paced && (done & 3) == 0) asm volatile("bar.sync 1, %0;" ::"r"(present * 32) : "memory");
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
        }
      if constexpr (FMT != 16) {
        const float unit = power_of_two(top_scale - 14);
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][nt][e] *= unit;
      }
      if (from_start && to_end) {
        finish(std::integral_constant<int, KS>{}, 0, o, cur.b, cur.hc, m, l);
      } else {
        const bool last = i == g1;           // every stage has been read, and no copy is under way
        float* part = last ? ring_of(warp) : a.part + (long long)me * kPart;
        __syncwarp();
#pragma unroll
        for (int t = 0; t < KS; ++t) store_tile(part, t, o[t]);
        store_sums(part, m, l);
        if (lane == 0) parts[2 * warp + last] = Part{part, i - cur.t, i - cur.t + cur.tiles, cur.b, cur.hc};
      }
      --cur.t;                               // the loop above left it one past the pair's last tile
      advance(cur);
    }
  }

  // ---- pairs in several ranges: first this CTA's parts of them, then those that it completes, of all CTAs ----
  const int G0 = start_of(me0), G1 = start_of(me1);
  float* cta_parts = a.part + (long long)ctas * kWarps * kPart;       // of CTA c: 2 c (its first pair), 2 c + 1 (its last)
  Part cut[2];                               // the pair that began before this CTA, the one that goes on behind it
  cut[0].at = cut[1].at = nullptr;
  for (int round = 0;; ++round) {
    __syncthreads();
    const Part mine = parts[lane];
    uint32_t left = __ballot_sync(0xffffffffu, mine.at != nullptr);
    int item = warp;                         // of KS accumulator tiles a pair, one a warp in turn
    while (left) {
      const Part pair = parts[__ffs(left) - 1];
      const uint32_t run = __ballot_sync(0xffffffffu, mine.at != nullptr && mine.begin == pair.begin);
      left &= ~run;
      const bool here = round == 1 || (pair.begin >= G0 && pair.end <= G1);
      if (!here) cut[pair.begin < G0 ? 0 : 1] = pair;
      for (; item < KS; item += kWarps) {
        float acc[1][NT][4], M[NT][2], L[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[0][nt][e] = 0.f;
            M[nt][e & 1] = -INFINITY;
            L[nt][e & 1] = 0.f;
          }
#pragma unroll 1
        for (uint32_t u = run; u;) {         // four parts in flight
          const float* at[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            at[k] = u ? parts[__ffs(u) - 1].at : nullptr;
            u &= u - 1;
          }
          add_parts(at, item, acc, M, L);
        }
        if (here) {
          finish(std::integral_constant<int, 1>{}, item, acc, pair.b, pair.hc, M, L);
        } else {
          float* part = cta_parts + ((long long)cta * 2 + (pair.begin < G0 ? 0 : 1)) * kPart;
          store_tile(part, item, acc[0]);
          if (item == 0) store_sums(part, M, L);
        }
      }
      item -= KS;
    }
    if (round == 1 || (!cut[0].at && !cut[1].at)) break;
    __threadfence();
    __syncthreads();
    if (tid < 2) {
      const Part p = tid ? cut[1] : cut[0];
      int n = 0;
      if (p.at) {
        const int c0 = worker_of(p.begin) / active, c1 = worker_of(p.end - 1) / active;
        int* count = a.counters + p.b * Hc + p.hc;
        if (atomicAdd(count, 1) == c1 - c0) {
          *count = 0;
          n = c1 - c0 + 1;
        }
        flag[2 + tid] = c0;
      }
      flag[tid] = n;
    }
    __syncthreads();
    const int n0 = flag[0], n1 = flag[1];
    if (n0 + n1 == 0) break;
    __threadfence();
    auto part_of = [&](int c, int begin) { return cta_parts + ((long long)c * 2 + (start_of(c * active) > begin ? 0 : 1)) * kPart; };
    if (n0 + n1 <= 8) {
      if (warp == 0) {
        const int x = lane < n0 ? 0 : 1;
        Part p = x ? cut[1] : cut[0];
        p.at = lane < n0 + n1 ? part_of(flag[2 + x] + lane - (x ? n0 : 0), p.begin) : nullptr;
        parts[lane] = p;
      }
      continue;
    }
    // parts of more CTAs: every warp first sums its share of them into its ring (a part's loads take a microsecond)
    if (tid < 32) parts[tid].at = nullptr;
    __syncthreads();
#pragma unroll 1
    for (int x = 0; x < 2; ++x) {
      const int n = x ? n1 : n0;
      if (warp >= n) continue;
      Part p = x ? cut[1] : cut[0];
      float* part = ring_of(warp) + x * kPart;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[nt][e & 1] = -INFINITY;
          l[nt][e & 1] = 0.f;
#pragma unroll
          for (int t = 0; t < KS; ++t) o[t][nt][e] = 0.f;
        }
#pragma unroll 1
      for (int k = warp; k < n; k += kWarps) add_part(part_of(flag[2 + x] + k, p.begin), o, m, l);
#pragma unroll
      for (int t = 0; t < KS; ++t) store_tile(part, t, o[t]);
      store_sums(part, m, l);
      p.at = part;
      if (lane == 0) parts[2 * warp + x] = p;
    }
  }
  // beside the launch of the shared prefixes: this one is complete no sooner than that one, so the one that joins them finds
  // both (one thread's wait is enough; one of every CTA cost 64 rows behind two prefixes 4 us of 54)
  if (a.groups > 0 && cta == 0 && tid == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Rows of a batch with shared prefixes: what the decode launch left of a row and the parts of its group's prefix.
struct MergeArgs {
  const float *own_o, *own_ml, *pre_o, *pre_ml;     // pre: [group][tile pair][key head][part][256 rows][D and 2]
  const int *cu_rows, *shared;
  __nv_bfloat16* out;
  long long ldo;
  int B, Hq, Hkv, groups, most_shared, pairs, parts, blocks_per_part;
  unsigned int* status;
};

// A warp a row (sequence, query head): 4 or 2 channels a lane, all parts' loads in flight together.  Bound by latency: 64
// rows of 32 heads with 9 parts are 10 MB out of the L2 cache.
template <int D>
__global__ void __launch_bounds__(256) scored_merge_kernel(const MergeArgs a) {
  constexpr int kC = D / 32;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.B * a.Hq) return;
  const int b = row / a.Hq, head = row - b * a.Hq, share = a.Hq / a.Hkv, hk = head / share;
  float acc[kC];
#pragma unroll
  for (int c = 0; c < kC; ++c) acc[c] = a.own_o[(long long)row * D + lane * kC + c];
  float M = a.own_ml[row * 2], L = a.own_ml[row * 2 + 1];
  if (M == -INFINITY) {          // no key of it has a weight (L is zero), or no score is a number (nor is L)
#pragma unroll
    for (int c = 0; c < kC; ++c) acc[c] = 0.f;
  }
  const int per = 128 / share;                               // sequences of a 128-row tile of the prefix kernel
  const int g = group_of(a.cu_rows, a.groups, b, a.pairs * 2 * per, a.status);
  if (g >= 0) {
    // the parts that the prefix launch wrote: as many as its keys fill
    const int blocks = (min(a.shared[g], a.most_shared) + 127) >> 7;
    const int np = (blocks + a.blocks_per_part - 1) / a.blocks_per_part;
    const int r = b - a.cu_rows[g], tile = r / per, in_tile = (r - tile * per) * share + head - hk * share;
    const long long at = ((((long long)g * a.pairs + (tile >> 1)) * a.Hkv + hk) * a.parts) * 256 + (tile & 1) * 128 + in_tile;
    for (int i0 = 0; i0 < np; i0 += 8) {
      float2 v[8];
      float p[8][kC];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long from = at + (long long)min(i0 + i, np - 1) * 256;
        v[i] = *reinterpret_cast<const float2*>(a.pre_ml + from * 2);
#pragma unroll
        for (int c = 0; c < kC; ++c) p[i][c] = a.pre_o[from * D + lane * kC + c];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= np || v[i].y == 0.f) continue;   // a part of weight zero may hold anything
        if (v[i].x == -INFINITY) {                     // no score is a number
          L += v[i].y;
          continue;
        }
        const float top = fmaxf(M, v[i].x), f = M == -INFINITY ? 0.f : ex2(M - top), w = ex2(v[i].x - top);
        M = top;
        L = fmaf(w, v[i].y, L * f);
#pragma unroll
        for (int c = 0; c < kC; ++c) acc[c] = fmaf(w, p[i][c], acc[c] * f);
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  __nv_bfloat16* to = a.out + (long long)b * a.ldo + (long long)head * D + lane * kC;
#pragma unroll
  for (int c = 0; c < kC; c += 2) *reinterpret_cast<uint32_t*>(to + c) = us::pack_bf(acc[c] * inv, acc[c + 1] * inv);
}

template <int D, int FMT, int NT>
int launch(const DecodeArgs& a, int ctas, cudaStream_t stream) {
  const size_t bytes = shared_bytes<D, FMT, NT>();
  static_assert(shared_bytes<D, FMT, NT>() <= 232448, "shared memory");
  US_CUDA_CHECK((us::allow_shared<scored_decode_kernel<D, FMT, NT>>((int)bytes)));
  US_CUDA_CHECK(us::launch_pdl(scored_decode_kernel<D, FMT, NT>, dim3(ctas), dim3(Shape<D, FMT, NT>::kWarps * 32), bytes, stream, a));
  return US_OK;
}

}  // namespace

// Bytes of the partial results of a launch on the current device: a part for each of the 8 warps (of 16 heads) or 16 warps
// (of 8), two for each CTA.  (Its counters: B * Hkv * ceil(Hq / Hkv / 16) int32.)
US_API long long us_scored_decode_scratch(int D) {
  int sms = 0;
  if (us::sm_count(&sms) != cudaSuccess) return -1;
  const long long two = (8 + 2) * 2, one = (16 + 2) * 1;
  return (long long)sms * (two > one ? two : one) * (D * 8 + 16) * (long long)sizeof(float);
}

// q [B, Hq, D] bf16 (row pitch ldq); pages [pages, page, Hkv, D] bf16 or integer codes with scales (bits 8, 4; 16: bf16);
// table [B, max_pages], lens [B], starts [B] or null.  scratch, counters: see above; counters are zero before the first
// call and left zero; calls that share them are ordered on the device.  groups > 0: the keys below min(shared[g],
// most_shared) of rows [cu_rows[g], cu_rows[g + 1]) are in pre_o / pre_ml by us_scored_prefix (with the same numbers), the
// launch before this one on the stream, and own_o, own_ml ([B][Hq][D and 2] floats) take the rest until both are joined.
US_API int us_scored_decode(const void* q, long long ldq, const void* kc, const void* vc, const void* ks, const void* vs,
                            const int* table, int max_pages, const int* lens, const int* starts, void* out, long long ldo,
                            void* scratch, int* counters, int B, int Hq, int Hkv, int D, int bits, int pages, int page,
                            int window, float scale, float cap, const float* slopes, int groups, const int* cu_rows,
                            const int* shared, int most_shared, const float* pre_o, const float* pre_ml, float* own_o,
                            float* own_ml, int pairs, int parts, int blocks_per_part, void* stream_) {
  US_REQUIRE(B >= 0 && B <= kMaxSeqs && (D == 64 || D == 128) && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0);
  if (B == 0) return US_OK;
  US_REQUIRE(q && kc && vc && table && lens && out && scratch && counters && max_pages >= 1 && pages >= 1 && page >= 1);
  US_REQUIRE(bits == 16 || ((bits == 8 || bits == 4) && ks && vs && page % 2 == 0 && (((uintptr_t)ks | (uintptr_t)vs) % 4) == 0));
  US_REQUIRE((long long)pages * page <= 0x7fffffffLL && window >= 0 && cap >= 0.f);
  if ((long long)pages * page * Hkv * (D * bits / 128) >= 0xffffffffLL) return US_ERR_LIMIT;   // places are 32 bits of 16 bytes
  // the tile list of the longest sequences that the page table holds is counted in 31 bits
  if ((((long long)max_pages * page + 31) / 32 + 1) * B > 0x7fffffffLL / (Hkv * ((Hq / Hkv + 15) / 16))) return US_ERR_LIMIT;
  US_REQUIRE((ldq % 8) == 0 && (ldo % 2) == 0 && (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) % 16) == 0 &&
             ((uintptr_t)out % 4) == 0);
  const int share = Hq / Hkv;
  if (groups > 0) US_REQUIRE(cu_rows && shared && pre_o && pre_ml && own_o && own_ml && pairs >= 1 && parts >= 1 && blocks_per_part >= 1 && share <= 128 &&
                             window == 0 && !starts && most_shared >= 0 && (long long)most_shared <= (long long)parts * blocks_per_part * 128);
  DecodeArgs a = {};
  a.q = (const __nv_bfloat16*)q;
  a.kc = (const uint8_t*)kc;
  a.vc = (const uint8_t*)vc;
  a.ks = (const __nv_bfloat16*)ks;
  a.vs = (const __nv_bfloat16*)vs;
  a.table = table;
  a.lens = lens;
  a.starts = starts;
  a.out = (__nv_bfloat16*)out;
  int sms = 0;
  US_CUDA_CHECK(us::sm_count(&sms));
  a.part = (float*)scratch;
  a.counters = counters;
  a.slopes = slopes;
  a.ldq = ldq;
  a.ldo = ldo;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.chunks = (share + 15) / 16;
  a.max_pages = max_pages;
  a.pages = pages;
  a.page = page;
  a.shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1;
  a.window = window;
  const float kLog2e = 1.4426950408889634f;
  a.scale_log2 = scale * kLog2e;
  a.cap_log2 = cap * kLog2e;
  a.scale_cap = cap > 0.f ? 2.f * scale * kLog2e / cap : 0.f;
  a.groups = groups;
  a.most_shared = most_shared;
  a.most_rows = pairs * 2 * (128 / share);
  a.cu_rows = cu_rows;
  a.shared = shared;
  a.own_o = own_o;
  a.own_ml = own_ml;
  a.status = us_status_ptr();
  a.magic = bits == 8 ? 0x64646464u : 0x54005400u;
  cudaStream_t stream = (cudaStream_t)stream_;
  int rc = US_ERR_UNSUPPORTED;
#define US_SCORED(DD, F)                                                                   \
  if (D == DD && bits == F) rc = share <= 8 ? launch<DD, F, 1>(a, sms, stream) : launch<DD, F, 2>(a, sms, stream)
  US_SCORED(64, 16);
  US_SCORED(64, 8);
  US_SCORED(64, 4);
  US_SCORED(128, 16);
  US_SCORED(128, 8);
  US_SCORED(128, 4);
#undef US_SCORED
  if (rc || groups == 0) return rc;
  MergeArgs m;
  m.own_o = own_o;
  m.own_ml = own_ml;
  m.pre_o = pre_o;
  m.pre_ml = pre_ml;
  m.cu_rows = cu_rows;
  m.shared = shared;
  m.out = (__nv_bfloat16*)out;
  m.ldo = ldo;
  m.B = B;
  m.Hq = Hq;
  m.Hkv = Hkv;
  m.groups = groups;
  m.most_shared = most_shared;
  m.pairs = pairs;
  m.parts = parts;
  m.blocks_per_part = blocks_per_part;
  m.status = a.status;
  // plain stream order: both launches before it are complete (the decode launch does not wait for the prefix's)
  const int rows = B * Hq;
  if (D == 64) scored_merge_kernel<64><<<(rows + 7) / 8, 256, 0, stream>>>(m);
  else scored_merge_kernel<128><<<(rows + 7) / 8, 256, 0, stream>>>(m);
  US_LAUNCH_CHECK();
  return US_OK;
}
