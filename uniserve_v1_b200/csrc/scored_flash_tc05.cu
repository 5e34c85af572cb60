// Softmax attention of prompts whose scores are capped by a tanh, biased by distance, or masked by a window, a prefix
// or documents; and the part of a decode batch's attention that a shared prefix has (scored_decode.cu has the rest).
//
//   s = scale q.k_j;  s = cap tanh(s / cap);  s -= slope |p - j|;  out = sum_j e^s v_j / sum_j e^s over visible j
//
// A CTA has two tiles of 128 rows, each row one of a few query heads at one position, and walks the 128-key blocks that any
// of them sees; the tensor pipe alternates between the tiles, so one tile's softmax runs under the other's products.  S_X = Q_X K^T and O_X += P_X V are
// tcgen05 products with S, P and O in tensor memory (P over the first half of S), operands by TMA, one thread a row in
// the softmax (the layout of flash_attn2_tc05.cu).  What differs:
//
// * Blocks.  Before it starts a CTA writes down, one bit a block and tile, which blocks its rows see, from positions,
//   window, prefix and, for documents, the smallest and largest document of each block; all roles walk these bits.
//   A tile that does not see a block that the other one does takes no part in it.
// * Masks.  In a block that not all rows of a warp see whole, a row's visible keys are 128 bits: intervals by
//   arithmetic, documents by a ballot per distinct document among the warp's rows.
// * Cap.  tanh costs the special-function unit, which the exponentials alone fill as long as the tensor pipe is
//   busy (16,384 of either a block and tile, 1024 cycles), as much again or, by e^(2y) and a reciprocal, twice.  So
//   cap tanh(s / cap) is an odd polynomial of degree seven in s on the FMA pipe, two scores an instruction, five
//   instructions a pair (off by at most 3.6e-6 cap for |s| <= 0.75 cap; fitted here by weighted least squares to
//   tanh's values); a warp that meets a larger score in a block takes the exponential form there.
// * Bias.  Keys on one side of a row are a line in j, added within the polynomial's last multiply-add; a block
//   with keys on both sides takes magnitudes.
// * Values behind the last key of a sequence (of a shared prefix: of the longest row) are put to zero in shared memory before
//   their product: they belong to another sequence, or to nobody, and 0 x NaN is NaN.
//
// A shared prefix: rows of a tile are (sequence, query head of the key head) pairs of one group, the keys come through
// the page list of the group's first row (or packed), split into `parts` of the blocks; unnormalised outputs, maxima and
// sums go to the workspace.  Every wait is bounded.
//
// Bound by the softmax: 3,200 to 3,500 cycles a block of two tiles, 2,048 of them products.  4096 causal rows of 32 / 4 heads
// of 128: 133 to 143 us with or without a cap (0.97 - 1.03 PFLOP/s), 148 with a cap and a bias; documents of 600 keys in 8,192
// rows: 107 - 114 us, a third of it starts and ends of CTAs.  Caps above 55.45 have no fixed base and take the general form in
// every block, an exponential and a reciprocal more a score: 300 us at 56 and at 100, 139 at 55.  A capped prefix of integer
// pages takes it too (FP16 weights need a maximum).
#include <type_traits>
#include "include/us_common.cuh"
#include "include/us_flash.cuh"
#include "include/us_tc05.cuh"
#include "include/us_tmap.h"

namespace {

using namespace flash;

constexpr int kBM = 128, kBN = 128;
constexpr int kHalf = 128 * 128;              // bytes of 64 columns of a tile
constexpr float kRescaleThreshold = 8.f;      // log2 units
constexpr int kMaxBlocks = 8192;              // key blocks of a sequence
constexpr int kWords = kMaxBlocks / 32;
constexpr int kThreads = 384;                 // two warpgroups of softmax rows; loads, products and two idle warps
constexpr float kPolyReach = 0.75f;           // of the cap
constexpr float kLog2e = 1.4426950408889634f;

struct ScoredArgs {
  const int *cu_q, *cu_k;
  __nv_bfloat16* out;
  long long ldo;
  int Tq, Tk, Hq, Hkv, causal, window;
  const int *docs, *prefix;
  const int2* ranges;                         // smallest and largest document of block j of sequence s at cu_k[s] / 128 + s + j
  const float* slopes;
  float scale_log2;
  float poly[4], reach, scale_cap, cap_log2;  // cap: x = s (p0 + p1 s^2 + ...) where |s| <= reach
  int pack;                                   // prompts: log2 of the query heads in a tile
  float base;                                 // what stands for every row's maximum under a small cap
  // shared prefixes
  const int *table, *lens, *cu_rows, *shared;
  const float* q_back;                        // FP16 operands (quant_pages.cu): factors of the rows of Q,
  const int2* exps;                           // and exponent fields of K and V [groups * Hkv]
  int key_stride;                             // > 0: packed keys, those of group g from row g * key_stride on
  int most_shared;                            // keys of a prefix at most
  int max_pages, pages, page, batch, pairs, parts, blocks_per_part;
  int n, max_q, max_k;                        // sequences, the longest one's rows and keys
  int fill;                                   // zeros in the output rows of no sequence
  float *part_o, *part_ml;
  unsigned int* status;
};

__device__ __forceinline__ unsigned long long add2_rm(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rm.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// The largest of two, three; NaN if one of them is.
__device__ __forceinline__ float max2_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^t for two arguments in [-126, 128) on the FMA pipe (flash_attn2_tc05.cu): relative error 8.6e-5.  (It takes NaN for -126.)
__device__ __forceinline__ void ex2_poly2(float t0, float t1, float& p0, float& p1) {
  const float kMagic = 12582912.f;
  const unsigned long long x = pack2(fmaxf(t0, -126.f), fmaxf(t1, -126.f));
  const unsigned long long tt = add2_rm(x, pack2(kMagic, kMagic));
  const unsigned long long fr = fma2(add2(tt, pack2(-kMagic, -kMagic)), pack2(-1.f, -1.f), x);
  unsigned long long p = fma2(fr, pack2(0.07706704f, 0.07706704f), pack2(0.22764499f, 0.22764499f));
  p = fma2(p, fr, pack2(0.69511676f, 0.69511676f));
  p = fma2(p, fr, pack2(1.f, 1.f));
  float q0, q1, u0, u1;
  unpack2(p, q0, q1);
  unpack2(tt, u0, u1);
  p0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(u0) << 23));
  p1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(u1) << 23));
}

__device__ __forceinline__ float power_of_two(int field) { return __uint_as_float((uint32_t)min(max(field, 0), 254) << 23); }
// bits [lo, hi) of 32
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (0xffffffffu >> (32 - (hi - lo))) << lo;
}

// The blocks that a CTA walks, the last first: under a distance bias a row's largest scores are beside it, and a maximum
// that is found first makes no output be scaled again.
struct Blocks {
  const uint32_t* bits;     // [kWords] of tile A, then of tile B
  int word;
  uint32_t left;
  __device__ __forceinline__ Blocks(const uint32_t* b, int words) : bits(b), word(words - 1), left(words > 0 ? b[words - 1] | b[kWords + words - 1] : 0) {}
  // the next block, and whether the tiles take part in it; -1 at the end
  __device__ __forceinline__ int next(bool& a, bool& b) {
    while (left == 0) {
      if (--word < 0) return -1;
      left = bits[word] | bits[kWords + word];
    }
    const int i = 31 - __clz(left);
    left ^= 1u << i;
    a = (bits[word] >> i) & 1u;
    b = (bits[kWords + word] >> i) & 1u;
    return word * 32 + i;
  }
};

// MODE 0: prompts.  1: shared prefixes.  2: prompts of few rows, the keys in parts.
// FIXED: no running maximum (see set_rules).  EMU: which of every eight exponential pairs go to the polynomial.
template <int kD, bool CAP, bool BIAS, bool FIXED, int MODE, uint32_t EMU>
__global__ void __launch_bounds__(kThreads, 1)
scored_flash_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const ScoredArgs a) {
  if (MODE != 1) {
    US_PDL_PROLOGUE();
  } else {       // the launch behind this one (scored_decode.cu) does not wait: it may start once what both read is there
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  constexpr bool PROMPT = MODE != 1, PARTS = MODE != 0;
  constexpr int kHalves = kD / 64, kTile = kHalves * kHalf;
  constexpr int kTmaWarp = 8, kMmaWarp = 9;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int share = a.Hq / a.Hkv;
  int seq, h = 0, hk, q0, q_start = 0, q_len, k_start, kv_len, shift = 0, per = kBM, pre = 0, part = 0;
  long long prow0 = 0;
  if constexpr (PROMPT) {
    seq = blockIdx.y;
    part = MODE == 2 ? (int)blockIdx.x % a.parts : 0;
    h = (MODE == 2 ? (int)blockIdx.x / a.parts : (int)blockIdx.x) << a.pack;      // the first of the tile's heads
    hk = h / share;
    per = kBM >> a.pack;
    // under a causal mask the last rows walk the most blocks: those of all heads and sequences start first
    q0 = (a.causal ? (int)gridDim.z - 1 - (int)blockIdx.z : (int)blockIdx.z) * 2 * per;
    const int rows_from = a.cu_q[0], rows_to = a.cu_q[a.n];      // (of all sequences; fetched beside the others)
    q_start = a.cu_q[seq];
    q_len = min(a.cu_q[seq + 1], a.Tq) - q_start;
    k_start = a.cu_k[seq];
    kv_len = min(a.cu_k[seq + 1] - k_start, a.Tk - k_start);
    shift = (a.cu_k[seq + 1] - k_start) - (a.cu_q[seq + 1] - q_start);
    if (a.prefix) pre = max(0, min(a.prefix[seq], kv_len));
    // rows and keys past what the host was told of the longest sequence, or past the tensors: some or all are left out
    bool short_of = q_len > (int)gridDim.z * 2 * per || kv_len > a.max_k || a.cu_q[seq + 1] > a.Tq || a.cu_k[seq + 1] > a.Tk;
    if (q_start < 0 || k_start < 0) {
      short_of = true;
      q_len = 0;
    }
    if (MODE == 2) {
      short_of |= q_len > a.max_q;
      q_len = min(q_len, a.max_q);
    }
    if (short_of && tid == 0) us_dev_fail(a.status, US_DEV_BOUNDS);
    if (a.fill && warp == kThreads / 32 - 1) {      // a warp that has nothing else to do; a share of those rows a CTA
      const int before = max(0, min(rows_from, a.Tq)), end = max(before, min(rows_to, a.Tq));
      const long long ctas = (long long)gridDim.x * gridDim.y * gridDim.z;
      for (long long i = blockIdx.x + (long long)gridDim.x * (blockIdx.y + (long long)gridDim.y * blockIdx.z); i < before + a.Tq - end; i += ctas) {
        uint4* row = reinterpret_cast<uint4*>(a.out + (i < before ? i : end + i - before) * a.ldo);
        for (int c = lane; c < a.Hq * (kD / 8); c += 32) row[c] = make_uint4(0, 0, 0, 0);
      }
    }
  } else {
    seq = blockIdx.z;
    hk = blockIdx.y % a.Hkv;
    const int pair = blockIdx.y / a.Hkv;
    part = blockIdx.x;
    per = kBM / share;
    q_start = a.cu_rows[seq];                                   // sequences of the group
    q_len = q_start < 0 ? 0 : min(a.cu_rows[seq + 1], a.batch) - q_start;      // (see group_of in scored_decode.cu)
    q0 = pair * 2 * per;
    k_start = seq * a.key_stride;
    kv_len = min(a.shared[seq], a.most_shared);
    if (part == 0 && blockIdx.y == 0 && q_len > 0) {
      // a prefix past the page lists or longer than told: what is left of it is the rows' own
      bool bad = a.shared[seq] > a.most_shared;
      if (a.key_stride > 0) {                  // packed keys: pages outside the cache were left out of them
        for (int pi = threadIdx.x; pi * a.page < kv_len; pi += kThreads)
          bad |= (unsigned)a.table[(long long)q_start * a.max_pages + pi] >= (unsigned)a.pages;
      }
      if (bad) us_dev_fail(a.status, US_DEV_BOUNDS);
    }
    prow0 = ((((long long)seq * a.pairs + pair) * a.Hkv + hk) * a.parts + part) * (2 * kBM);
  }
  if (q0 >= q_len) return;
  // where a row's part is: [part][sequence][row][head]
  auto part_row = [&](int row, int head) -> long long {
    return ((((long long)part * a.n + seq) * a.max_q + row) * a.Hq) + head;
  };
  kv_len = max(kv_len, 0);
  int nb = kv_len / kBN + (kv_len % kBN != 0), jb = 0;
  if constexpr (MODE == 1) {
    jb = part * a.blocks_per_part;
    nb = min(nb - jb, a.blocks_per_part);                       // kMaxBlocks at most
    if (nb <= 0) return;                                        // such a part is not read
  } else {
    nb = min(nb, kMaxBlocks);
  }

  int first_known = -1;
  if constexpr (PROMPT) {
    const int last = min(q0 + 2 * per, q_len) - 1 + shift;     // position of the last row
    if (nb > 0 && a.causal && last >= 0 && (!a.docs || pre <= last + 1)) first_known = max(last, pre - 1) / kBN;
    else if (nb > 0 && !a.causal && !a.docs) first_known = nb - 1;
    if (MODE == 2) first_known = -1;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                  // two tiles
  uint8_t* sK = smem + 2 * kTile;      // two stages
  uint8_t* sV = smem + 4 * kTile;      // two stages
  uint64_t* bars = (uint64_t*)(smem + 6 * kTile);
  uint64_t* q_full = bars;
  uint64_t* kv_full = bars + 1;        // [2]: V of a block and K of the next one
  uint64_t* kv_empty = bars + 3;       // [2]
  uint64_t* s_full = bars + 5;         // [2] by tile, like the next two
  uint64_t* p_full = bars + 7;
  uint64_t* o_full = bars + 9;
  uint32_t* tmem_slot = (uint32_t*)(bars + 11);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* taken = (int*)(tmem_slot + 2);  // [2]: blocks of each tile
  uint32_t* bits = tmem_slot + 4;      // [2][kWords]

  if (tid == 0) {
    tc::mbar_init(q_full, 2);          // Q, and the first block's K
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 128);
      tc::mbar_init(&o_full[i], 1);
      taken[i] = 0;
    }
    *abort_flag = 0;
    tc::mbar_fence_init();
    // Q is on its way while the blocks are looked up, and so is the first block's K where it is known: the last block,
    // or that of the last row's own key (which is of its document), or the one of the prefix's end
    tc::mbar_expect_tx(q_full, PROMPT ? 2 * kTile : 2 * kHalves * per * share * 128);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        uint8_t* to = sQ + x * kTile + hf * kHalf;
        tc::tma_load_3d(to, &tmQ, q_full, 64 * hf, PROMPT ? h : hk * share, q_start + q0 + x * per);
      }
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  __syncthreads();
  if (first_known >= 0 && tid == 0) {
    tc::mbar_expect_tx(q_full, kTile);
#pragma unroll
    for (int hf = 0; hf < kHalves; ++hf)
      tc::tma_load_2d(sK + hf * kHalf, &tmK, q_full, hk * kD + 64 * hf, k_start + first_known * kBN);
  }
  // ---- which blocks the tiles see ----
  const int words = (nb + 31) / 32;
  const int2* ranges = nullptr;
  if constexpr (PROMPT) {
    if (a.docs) ranges = a.ranges + (k_start / kBN + seq);
  }
  for (int w = warp; w < 2 * words; w += kThreads / 32) {
    const int x = w >= words, wi = w - x * words;
    const int j = wi * 32 + lane;
    bool see = j < nb;
    if constexpr (PROMPT) {
      const int r0 = q0 + x * per, r1 = min(r0 + per, q_len) - 1;          // the tile's rows
      const int pa = r0 + shift, pb = r1 + shift;                         // and their positions
      const int k0 = j * kBN, k1 = min(k0 + kBN, kv_len);
      see &= r0 < q_len;
      if (MODE == 2) see &= j / a.blocks_per_part == part;
      bool by_place = !a.causal || k0 <= pb;
      if (a.window > 0) by_place &= k1 - 1 > pa - a.window;
      see &= by_place || k0 < pre;
      if (see && ranges) {
        see = pb >= 0;
        if (see) {
          const int2 d0 = ranges[min(max(pa, 0), kv_len - 1) / kBN], d1 = ranges[min(pb, kv_len - 1) / kBN], d = ranges[j];
          see = d.x <= max(d0.y, d1.y) && d.y >= min(d0.x, d1.x);
        }
      }
    } else {
      see &= q0 + x * per < q_len;
    }
    const uint32_t got = __ballot_sync(0xffffffffu, see);
    if (lane == 0) {
      bits[x * kWords + wi] = got;
      if (got) atomicAdd(&taken[x], __popc(got));
    }
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int taken_a = taken[0], taken_b = taken[1];

  if (PROMPT && tid < 2 * kBM) {    // rows that see nothing
    const int x = tid >> 7, row = q0 + (tid >> a.pack), head = h + (tid & ((1 << a.pack) - 1));
    if ((x ? taken_b : taken_a) == 0 && row < q_len) {
      if constexpr (MODE == 2) {
        *reinterpret_cast<float2*>(a.part_ml + part_row(row, head) * 2) = make_float2(-INFINITY, 0.f);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(a.out + (long long)(q_start + row) * a.ldo + (long long)head * kD);
        for (int i = 0; i < kD / 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
      }
    }
  }

  // 384 threads are launched with 168 registers each (64,512); a row of scores wants more, the other roles less
  // (256 x 208 + 128 x 80 = 63,488)
  if (taken_a + taken_b == 0) {        // nothing is seen: Q has to have landed before the CTA ends
    if (tid == 0) {
      if (first_known < 0) tc::mbar_arrive(q_full);
      if (!tc::mbar_wait(q_full, 0, abort_flag)) us_dev_fail(a.status, US_DEV_TIMEOUT_FULL);
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kTmaWarp) {
      // ---------------------------------------------------------------- loads --
      // The whole warp walks; lane 0 loads whole tiles, or every lane its page of a tile.
      const bool paged = MODE == 1 && a.key_stride == 0;
      const int rows_at_once = paged ? min(a.page, kBN) : kBN;
      const int loads = kBN / rows_at_once;
      auto row_of = [&](int j) -> int {      // first row of this lane's load of block j
        const int key = (jb + j) * kBN + lane * rows_at_once;
        if (!paged) return k_start + key;
        if (lane >= loads || key >= kv_len) return a.pages * a.page;      // out of the tensor: zeros
        const int pi = key / a.page;
        const int pg = a.table[(long long)q_start * a.max_pages + pi];
        if ((unsigned)pg >= (unsigned)a.pages) {
          us_dev_fail(a.status, US_DEV_BOUNDS);
          return a.pages * a.page;
        }
        return pg * a.page + (key - pi * a.page);
      };
      auto load_tile = [&](uint8_t* to, const CUtensorMap* m, uint64_t* bar, int row) {
        if (lane < loads) {
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf)
            tc::tma_load_2d(to + hf * kHalf + lane * rows_at_once * 128, m, bar, hk * kD + 64 * hf, row);
        }
      };
      Blocks walk(bits, words);
      bool ta, tb;
      int j = walk.next(ta, tb);
      int row = row_of(j);
      if (first_known < 0) {
        if (lane == 0) tc::mbar_expect_tx(q_full, kTile);
        __syncwarp();
        load_tile(sK, &tmK, q_full, row);
      } else if (j != first_known && lane == 0) {      // (does not happen: see first_known)
        us_dev_fail(a.status, US_DEV_BOUNDS);
      }
      for (int e = 0; j >= 0; ++e) {
        const int st = e & 1;
        const int jn = walk.next(ta, tb);
        const int row_n = jn >= 0 ? row_of(jn) : 0;
        // kv_empty[1] completes first after the first S products: K stage 0 is free again
        if (!__all_sync(0xffffffffu, tc::mbar_wait(&kv_empty[st], ((uint32_t)((e + 1) >> 1) & 1u) ^ 1u, abort_flag))) {
          if (lane == 0) {
            us_dev_fail(a.status, US_DEV_TIMEOUT_EMPTY);
            *abort_flag = 1;
          }
          break;
        }
        if (lane == 0) tc::mbar_expect_tx(&kv_full[st], jn >= 0 ? 2 * kTile : kTile);
        __syncwarp();
        load_tile(sV + st * kTile, &tmV, &kv_full[st], row);
        if (jn >= 0) load_tile(sK + (st ^ 1) * kTile, &tmK, &kv_full[st], row_n);
        j = jn;
        row = row_n;
      }
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------- products --
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort_flag));
      };
      const uint32_t fmt = MODE == 1 && a.q_back ? tc::kFmtF16 : tc::kFmtBF16;
      const uint32_t kIdescQK = tc::make_idesc(kBM, kBN, fmt, fmt, 0, 0), kIdescPV = tc::make_idesc(kBM, kD, fmt, fmt, 0, 1);
      const uint64_t dq = tc::smem_desc_kmajor_sw128(tc::smem_u32(sQ));
      const uint64_t dk = tc::smem_desc_kmajor_sw128(tc::smem_u32(sK));
      const uint64_t dv = tc::smem_desc_mnmajor_sw128(tc::smem_u32(sV), kHalf, 1024);
      const uint32_t q_lo = (uint32_t)dq, k_lo = (uint32_t)dk, v_lo = (uint32_t)dv;
      const uint32_t km_hi = (uint32_t)(dq >> 32), mn_hi = (uint32_t)(dv >> 32);
      auto issue_qk = [&](int x, int e) {
        const uint32_t qa = q_lo + (uint32_t)x * (kTile >> 4), kb = k_lo + (uint32_t)(e & 1) * (kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk >> 2) * (kHalf >> 4) + 2u * (uint32_t)(kk & 3);
          umma_f16_words(tmem_base + (uint32_t)x * kBN, qa + off, km_hi, kb + off, km_hi, kIdescQK, kk != 0);
        }
        umma_commit_elect(&s_full[x]);
      };
      auto issue_pv = [&](int x, int e, int n, int all) {      // n: blocks of this tile so far
        const uint32_t vb = v_lo + (uint32_t)(e & 1) * (kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_f16_ts_words(tmem_base + 256 + (uint32_t)x * kD, tmem_base + (uint32_t)x * kBN + kk * 8,
                            vb + (uint32_t)kk * (2048 >> 4), mn_hi, kIdescPV, (n | kk) != 0);
        if (n == all - 1) umma_commit_elect(&o_full[x]);
      };
      Blocks walk(bits, words);
      bool a0 = false, b0 = false, a1 = false, b1 = false;
      int j = walk.next(a0, b0), na = 0, nbb = 0;
      bool ok = warp_wait(q_full, 0);
      if (ok) {
        tc::tc_fence_after_sync();
        if (a0) issue_qk(0, 0);
        if (b0) issue_qk(1, 0);
        umma_commit_elect(&kv_empty[1]);
      }
      int v_end = kv_len;                // values from here on nobody sees
      if constexpr (MODE == 1) {         // a prefix may be longer than the rows that share it
        int most = 0;
        for (int r = q0 + lane; r < min(q0 + 2 * per, q_len); r += 32) most = max(most, a.lens[q_start + r]);
        v_end = min(kv_len, __reduce_max_sync(0xffffffffu, most));
      }
      for (int e = 0; ok && j >= 0; ++e) {
        a1 = b1 = false;
        const int jn = walk.next(a1, b1);
        if (!warp_wait(&kv_full[e & 1], (uint32_t)(e >> 1) & 1u)) { ok = false; break; }
        const int there = v_end - (jb + j) * kBN;
        if (there < kBN) {               // the sequence ends in this block, or before it
          for (int r = max(there, 0) + (lane >> 3); r < kBN; r += 4)
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
              *reinterpret_cast<uint4*>(sV + (e & 1) * kTile + hf * kHalf + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          tc::fence_async_smem();
          __syncwarp();
        }
        if (a0) {
          if (!warp_wait(&p_full[0], (uint32_t)na & 1u)) { ok = false; break; }
          tc::tc_fence_after_sync();
          issue_pv(0, e, na++, taken_a);
        }
        if (a1) issue_qk(0, e + 1);
        if (b0) {
          if (!warp_wait(&p_full[1], (uint32_t)nbb & 1u)) { ok = false; break; }
          tc::tc_fence_after_sync();
          issue_pv(1, e, nbb++, taken_b);
        }
        if (b1) issue_qk(1, e + 1);
        umma_commit_elect(&kv_empty[e & 1]);
        j = jn;
        a0 = a1;
        b0 = b1;
      }
      if (!ok && lane == 0) {
        us_dev_fail(a.status, US_DEV_TIMEOUT_FULL);
        *abort_flag = 1;
      }
    }
  } else {
    {
      // -------------------------------------------------------------- softmax --
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int x = warp >> 2, r = (warp & 3) * 32 + lane;
      const uint32_t lane_addr = ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t s_tmem = tmem_base + (uint32_t)x * kBN + lane_addr;
      const uint32_t o_tmem = tmem_base + 256 + (uint32_t)x * kD + lane_addr;
      // the row: its position, its visible keys [lo, hi) and [0, pr), its document.  (Rows behind the last one have all that
      // of the last one, so that no warp takes another path for them: a ragged batch 219 -> 211 us.)
      int p, lo = 0, hi, pr = 0, doc = 0;
      float sl = 0.f;
      bool row_ok;
      [[maybe_unused]] int b_row = 0, head = 0;
      if constexpr (PROMPT) {
        const int row = q0 + x * per + (r >> a.pack);
        row_ok = row < q_len;
        p = min(row, q_len - 1) + shift;
        hi = a.causal ? min(kv_len, p + 1) : kv_len;
        if (a.window > 0) lo = max(0, p - a.window + 1);
        pr = pre;
        if (a.docs) {
          if (p >= 0 && p < kv_len) doc = a.docs[k_start + p];
          else hi = pr = 0;
        }
        if (BIAS) sl = a.slopes[h + (r & ((1 << a.pack) - 1))] * kLog2e;
      } else {
        row_ok = r < per * share && q0 + x * per + r / share < q_len;
        b_row = q_start + min(q0 + x * per + min(r / share, per - 1), q_len - 1);
        head = hk * share + r % share;
        p = a.lens[b_row] - 1;
        hi = min(kv_len, p + 1);
        if (BIAS) sl = a.slopes[head] * kLog2e;
      }
      if (BIAS && sl < 0.f) us_dev_fail(a.status, US_DEV_BOUNDS);      // (a fixed base has no room for scores that grow with distance)
      // FP16 operands: the scores' and the outputs' factors
      const bool half = MODE == 1 && a.q_back;
      // FP16 weights are held 2^14 times as large, 2^15 at most (the maximum may lag by one power of two): like those of the
      // integer pages' own decode they keep their bits down to 2^-28 of the largest, and end at 2^-39
      const float lift = half ? 14.f : 0.f, lag = half ? 1.f : kRescaleThreshold;
      float row_factor = 1.f, out_factor = 1.f;
      if (half) {
        const int2 top = a.exps[seq * a.Hkv + hk];
        out_factor = power_of_two(top.y);
        row_factor = a.q_back[(long long)b_row * a.Hq + head] * power_of_two(top.x);
      }
      const unsigned long long sc2 = pack2(a.scale_log2, a.scale_log2);
      unsigned long long c0 = 0, c1 = 0, c2 = 0, c3 = 0;
      if (CAP) {
        c0 = pack2(a.poly[0], a.poly[0]);
        c1 = pack2(a.poly[1], a.poly[1]);
        c2 = pack2(a.poly[2], a.poly[2]);
        c3 = pack2(a.poly[3], a.poly[3]);
      }
      // FIXED: what is taken for the maximum.  A row before the first key (p < 0, no causal mask) has all keys at least -p
      // away: that much bias is common to all.
      const float base = FIXED ? a.base - (BIAS && p < 0 ? sl * (float)-p : 0.f) : 0.f;
      float m_used = FIXED ? base : -INFINITY, m_next = m_used, l_sum = 0.f;
      Blocks walk(bits, words);
      int n = 0;
      bool ok = true;
      while (ok) {
        bool mine;
        int j;
        do {
          bool ta, tb;
          j = walk.next(ta, tb);
          mine = x ? tb : ta;
        } while (j >= 0 && !mine);
        if (j < 0) break;
        const int kbase = (jb + j) * kBN;
        // what of the block is visible to the row (looked up while the scores are computed)
        bool whole = (lo <= kbase && hi >= kbase + kBN) || pr >= kbase + kBN;
        if (PROMPT && ranges) {
          const int2 d = ranges[j];
          whole &= d.x == doc && d.y == doc;
        }
        const bool masked = __any_sync(0xffffffffu, !whole);
        uint32_t see[4];
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            see[c] = bits_between(lo - kbase - 32 * c, hi - kbase - 32 * c) | bits_between(0, pr - kbase - 32 * c);
          if (PROMPT && a.docs) {
            int kd[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int key = kbase + 32 * c + lane;
              kd[c] = key < kv_len ? a.docs[k_start + key] : 0;      // past the end: not visible by place
            }
            uint32_t left = 0xffffffffu;
            while (left) {                   // once for every document among the warp's rows
              const int d = __shfl_sync(0xffffffffu, doc, __ffs(left) - 1);
              const bool is = doc == d;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const uint32_t same = __ballot_sync(0xffffffffu, kd[c] == d);
                if (is) see[c] &= same;
              }
              left &= ~__ballot_sync(0xffffffffu, is);
            }
          }
        }
        if (!__all_sync(0xffffffffu, tc::mbar_wait(&s_full[x], (uint32_t)n & 1u, abort_flag))) { ok = false; break; }
        tc::tc_fence_after_sync();
        uint32_t v[kBN];
        auto fetch = [&]() {
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::tmem_ld32(s_tmem + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * c));
        };
        fetch();
        // O_X under another maximum.  It is still: this block's S was issued after the last block's product, by the same
        // thread.
        auto rescale = [&](float m_new) {
          const float alpha = m_used == -INFINITY ? 0.f : ex2f(m_used - m_new);
          if (n > 0) {
#pragma unroll 1
            for (int c = 0; c < kD; c += 32) {
              uint32_t w[32];
              tc::tmem_ld32(o_tmem + c, w);
              tc::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * alpha);
              tc::tmem_st32(o_tmem + c, w);
            }
          }
          l_sum *= alpha;
          m_used = m_new;
        };
        auto by_row = [&]() {                // FP16 operands were divided by powers of two
          if (MODE == 1 && half) {
#pragma unroll
            for (int i = 0; i < kBN; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * row_factor);
          }
        };
        tc::tmem_ld_wait();
        by_row();
        if (!FIXED && __any_sync(0xffffffffu, m_next - m_used > lag)) rescale(m_next);
        const int delta = p - kbase;
        // Whether the row's scores are cap's polynomial's.  (A comparison that a NaN fails: such a block takes the other
        // form, which passes it on.)
        bool poly = true;
        if (CAP) {
          float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 32; i += 2)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              big[c] = max3_abs(big[c], __uint_as_float(v[32 * c + i]), __uint_as_float(v[32 * c + i + 1]));
          poly = __all_sync(0xffffffffu, fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) <= a.reach);
        }
        // Keys on both sides of some row: magnitudes.  (Keys behind a row that it does not see need none: a causal row's bias
        // is a line.)
        const bool sides = BIAS && __any_sync(0xffffffffu, max(hi, pr) > p + 1 && delta > 0 && delta < kBN - 1);
        unsigned long long ls[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk[kBN / 2];
        auto weigh = [&](float t0, float t1, unsigned long long& l, bool emulate) -> uint32_t {
          float p0, p1;
          if (emulate) {
            ex2_poly2(t0, t1, p0, p1);
          } else {
            p0 = ex2f(t0);
            p1 = ex2f(t1);
          }
          l = add2(l, pack2(p0, p1));
          if (MODE == 1 && half) {
            const __half2 t = __floats2half2_rn(p0, p1);
            return *reinterpret_cast<const uint32_t*>(&t);
          }
          const __nv_bfloat162 t = __floats2bfloat162_rn(p0, p1);
          return *reinterpret_cast<const uint32_t*>(&t);
        };
        // One pass from scores to weights, so that the FMA pipe's polynomials and the special-function unit's exponentials
        // run side by side.  Without a fixed base the maximum is that of the blocks before: bf16 and FP32 have room for
        // what exceeds it, and the next block starts from this one's.
        bool through = false;
        auto pass = [&](auto with_mask) {
          constexpr bool MASK = decltype(with_mask)::value;
          const float less = FIXED ? -base : m_used == -INFINITY ? lift : lift - m_used;
          const float step = delta > 0 ? sl : -sl, at = BIAS ? fmaf(-sl, fabsf((float)delta), less) : less;
          unsigned long long b2[4];
          const unsigned long long st2 = pack2(2.f * step, 2.f * step);
#pragma unroll
          for (int c = 0; c < 4; ++c) b2[c] = BIAS ? pack2(fmaf(step, 32.f * c, at), fmaf(step, 32.f * c + 1.f, at)) : pack2(at, at);
          float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const unsigned long long s2 = pack2(__uint_as_float(v[32 * c + i]), __uint_as_float(v[32 * c + i + 1]));
              unsigned long long y;
              if (CAP) {
                const unsigned long long w = mul2(s2, s2);
                y = fma2(s2, fma2(fma2(fma2(c3, w, c2), w, c1), w, c0), b2[c]);
              } else {
                y = fma2(s2, sc2, b2[c]);
              }
              if (BIAS) b2[c] = add2(b2[c], st2);
              float t0, t1;
              unpack2(y, t0, t1);
              if (MASK) {
                if (!((see[c] >> i) & 1u)) t0 = -INFINITY;
                if (!((see[c] >> (i + 1)) & 1u)) t1 = -INFINITY;
              }
              if (!FIXED) mxs[c] = max3_nan(mxs[c], t0, t1);
              pk[16 * c + (i >> 1)] = weigh(t0, t1, ls[c], !MASK && ((EMU >> (((i >> 1) & 1) * 4 + c)) & 1u));
            }
          }
          if (!FIXED) {
            // of the maximum so far; a NaN fails the comparison, and the general form passes it on where the polynomial does not
            const float over = max2_nan(max2_nan(mxs[0], mxs[1]), max2_nan(mxs[2], mxs[3]));
            through = __all_sync(0xffffffffu, over <= (half ? lift + lag : 64.f));    // FP16 ends at 2^16
            m_next = fmaxf(m_used, m_used + (over - lift));
          } else {
            through = true;
          }
        };
        if ((FIXED || (!CAP && n > 0 && __all_sync(0xffffffffu, m_used > -INFINITY))) && poly && !sides) {
          if (masked) pass(std::true_type{});
          else pass(std::false_type{});
        }
        if (!through) {
          // the general form: scores in units of log2(e) less the base, masks, the maximum, weights
          if (!FIXED && !CAP && n > 0) {     // (the scores were weighed and are wanted again)
            fetch();
            tc::tmem_ld_wait();
            by_row();
          }
          const float at = (float)delta;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float s = __uint_as_float(v[32 * c + i]);
              if (CAP) {                     // tanh y = 1 - 2 / (1 + e^(2 y))
                s = fmaf(-2.f * a.cap_log2, rcpf(1.f + ex2f(s * a.scale_cap)), a.cap_log2 - base);
              } else {
                s *= a.scale_log2;
              }
              if (BIAS) s = fmaf(-sl, fabsf(at - (float)(32 * c + i)), s);
              if (masked && !((see[c] >> i) & 1u)) s = -INFINITY;
              v[32 * c + i] = __float_as_uint(s);
            }
          if (!FIXED) {
            float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 2)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                mxs[c] = max3(mxs[c], __uint_as_float(v[32 * c + i]), __uint_as_float(v[32 * c + i + 1]));
            const float m_new = fmaxf(m_used, fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3])));
            if (__any_sync(0xffffffffu, m_new > m_used)) rescale(m_new);
            m_next = m_used;
          }
          const float less = FIXED ? 0.f : m_used == -INFINITY ? -lift : m_used - lift;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            ls[c] = 0ull;
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              pk[16 * c + (i >> 1)] = weigh(__uint_as_float(v[32 * c + i]) - less, __uint_as_float(v[32 * c + i + 1]) - less, ls[c], false);
          }
        }
        {
          float s0, s1;
          unpack2(add2(add2(ls[0], ls[1]), add2(ls[2], ls[3])), s0, s1);
          l_sum += s0 + s1;
        }
        tc::tmem_st32(s_tmem, *reinterpret_cast<const uint32_t(*)[32]>(pk));
        tc::tmem_st32(s_tmem + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
        tc::tmem_st_wait();
        tc::tc_fence_before_sync();
        tc::mbar_arrive(&p_full[x]);
        ++n;
      }
      if (n > 0 || !ok) {
        if (ok && __all_sync(0xffffffffu, tc::mbar_wait(&o_full[x], 0, abort_flag))) {
          tc::tc_fence_after_sync();
          const float inv = MODE == 0 ? (l_sum == 0.f ? 0.f : 1.f / l_sum) : out_factor;
          const long long prow = prow0 + x * kBM;
          if (PARTS && row_ok) {
            const long long to = MODE == 2 ? part_row(q0 + x * per + (r >> a.pack), h + (r & ((1 << a.pack) - 1))) : prow + r;
            *reinterpret_cast<float2*>(a.part_ml + to * 2) = make_float2(m_used - lift, l_sum);
          }
          uint32_t all[kD];
#pragma unroll
          for (int c = 0; c < kD; c += 32) tc::tmem_ld32(o_tmem + c, *reinterpret_cast<uint32_t(*)[32]>(all + c));
          tc::tmem_ld_wait();
          // 64 bytes of every row at a time through shared memory (the tile's Q, which no product reads any more): eight
          // rows a store in place of 32 (4096 causal rows x 32 heads: 139 -> 133 us; short documents: 119 -> 111)
          constexpr int kPer = PARTS ? 16 : 32;      // channels
          const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_ok);
          uint8_t* lines = sQ + x * kTile + (warp & 3) * 2048;
          const int row0 = (warp & 3) * 32 + (lane >> 2);
#pragma unroll
          for (int c = 0; c < kD; c += kPer) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 piece;
              if constexpr (!PARTS) {
                us::Pack16 o;
#pragma unroll
                for (int k = 0; k < 8; ++k) o.b[k] = us::f2bf(__uint_as_float(all[c + i * 8 + k]) * inv);
                piece = o.u;
              } else {
                const uint32_t* w = all + c + i * 4;
                piece = make_uint4(__float_as_uint(__uint_as_float(w[0]) * inv), __float_as_uint(__uint_as_float(w[1]) * inv),
                                   __float_as_uint(__uint_as_float(w[2]) * inv), __float_as_uint(__uint_as_float(w[3]) * inv));
              }
              *reinterpret_cast<uint4*>(lines + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16) = piece;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (!((rows_ok >> (8 * i + (lane >> 2))) & 1u)) continue;
              const uint4 w = *reinterpret_cast<const uint4*>(lines + (8 * i + (lane >> 2)) * 64 + (((lane >> 3) ^ lane) & 3) * 16);
              const int at = row0 + 8 * i, at_row = q0 + x * per + (at >> a.pack), at_head = h + (at & ((1 << a.pack) - 1));
              if constexpr (MODE == 0)
                *reinterpret_cast<uint4*>(a.out + (long long)(q_start + at_row) * a.ldo + at_head * kD + c + (lane & 3) * 8) = w;
              else
                *reinterpret_cast<uint4*>(a.part_o + (MODE == 2 ? part_row(at_row, at_head) : prow + at) * kD + c + (lane & 3) * 4) = w;
            }
          }
        } else {
          us_dev_fail(a.status, US_DEV_TIMEOUT_ACC);
          *abort_flag = 1;
        }
      }
    }
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc::tmem_dealloc(tmem_base, 512);
  }
}

// Smallest and largest document of every 128-key block: a warp a block.
__global__ void __launch_bounds__(128) doc_ranges_kernel(const int* docs, const int* cu_k, int Tk, int2* ranges) {
  US_PDL_PROLOGUE();
  const int seq = blockIdx.y, j = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int start = cu_k[seq], end = min(cu_k[seq + 1], Tk);
  if (start < 0 || start + j * kBN >= end) return;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int k = start + j * kBN + 32 * c + lane;
    if (k < end) {
      const int d = docs[k];
      lo = min(lo, d);
      hi = max(hi, d);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) ranges[start / kBN + seq + j] = make_int2(lo, hi);
}

// Rows whose keys went in parts: a warp a row and head.
template <int D>
__global__ void __launch_bounds__(256) join_parts_kernel(const ScoredArgs a) {
  US_PDL_PROLOGUE();
  constexpr int kC = D / 32;
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.n * a.max_q * a.Hq, i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= rows) return;
  const int head = (int)(i % a.Hq), row = (int)(i / a.Hq % a.max_q), seq = (int)(i / a.Hq / a.max_q);
  const int start = a.cu_q[seq], end = a.cu_q[seq + 1], keys = a.cu_k[seq];
  if (min(start, keys) < 0 || row >= min(end, a.Tq) - start) return;      // such parts were not written
  float M = -INFINITY, L = 0.f, acc[kC] = {};
  for (int p0 = 0; p0 < a.parts; p0 += 4) {            // four parts' loads in flight
    float2 ml[4];
    float o[4][kC];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long at = (long long)min(p0 + k, a.parts - 1) * rows + i;
      ml[k] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
#pragma unroll
      for (int c = 0; c < kC; ++c) o[k][c] = a.part_o[at * D + lane * kC + c];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (p0 + k >= a.parts || ml[k].y == 0.f) continue;      // such a part may hold anything
      if (ml[k].x == -INFINITY) {                             // no score is a number
        L += ml[k].y;
        continue;
      }
      const float top = fmaxf(M, ml[k].x), f = M == -INFINITY ? 0.f : ex2f(M - top), w = ex2f(ml[k].x - top);
      M = top;
      L = fmaf(w, ml[k].y, L * f);
#pragma unroll
      for (int c = 0; c < kC; ++c) acc[c] = fmaf(w, o[k][c], acc[c] * f);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  __nv_bfloat16* to = a.out + (long long)(start + row) * a.ldo + (long long)head * D + lane * kC;
#pragma unroll
  for (int c = 0; c < kC; c += 2) *reinterpret_cast<__nv_bfloat162*>(to + c) = __floats2bfloat162_rn(acc[c] * inv, acc[c + 1] * inv);
}

size_t shared_bytes(int D) { return 6 * (size_t)(D / 64) * kHalf + 11 * 8 + 16 + 2 * kWords * 4 + 1024; }

void set_rules(ScoredArgs& a, float scale, float cap, const float* slopes) {
  a.scale_log2 = scale * kLog2e;
  a.slopes = slopes;
  if (cap > 0.f) {
    // tanh(y) ~ y (t0 + t1 y^2 + t2 y^4 + t3 y^6) for |y| <= 0.75, with y = s scale / cap; out of a reasonable range
    // of scale / cap the powers leave FP32's and the exponential form serves alone
    const double t[4] = {0.9999556, -0.33222756, 0.1257706, -0.0337779}, k = (double)scale / cap;
    double f = k * cap * (double)kLog2e;
    for (int i = 0; i < 4; ++i, f *= k * k) a.poly[i] = (float)(t[i] * f);
    const double mag = k < 0 ? -k : k;
    a.reach = mag > 1e-4 && mag < 1e4 ? (float)(kPolyReach / mag) : -1.f;
    a.scale_cap = (float)(2.0 * k * kLog2e);
    a.cap_log2 = cap * kLog2e;
    // Weights in [2^(-cap_log2 - base), 2^40], or, as a distance bias takes them down from there, in [.., 2^64]: 2^20 keys of
    // values up to 2^44 stay in FP32's range
    const float top = slopes ? 64.f : 40.f;
    a.base = a.cap_log2 > top ? a.cap_log2 - top : 0.f;
  }
}
// Caps under which weights need no maximum (those up to 55.45).  Without a bias the smallest weight is 2^-120 at least, and
// none is lost.  With one a row's own key weighs 2^-96 at least, so a key that FP32 ends above (2^-126) weighs under 2^-30 of it.
bool small_cap(const ScoredArgs& a) { return a.cap_log2 + a.base <= (a.slopes ? 96.f : 120.f); }

template <int D, bool CAP, bool BIAS, bool FIXED, int MODE>
int start(dim3 grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ScoredArgs& a, cudaStream_t stream) {
  // Exponentials on the FMA pipe: an eighth (no cap: 187 -> 179 us at 4096 causal rows x 32 heads), a quarter for 64-wide
  // heads, which have half the tensor work per exponential (275 -> 253 us); with a cap that pipe has enough to do (none:
  // 189 us, an eighth: 193).
  constexpr uint32_t kEmu = CAP ? 0u : D == 64 ? 0x21u : 0x01u;
  const size_t bytes = shared_bytes(D);
  US_CUDA_CHECK((us::allow_shared<scored_flash_kernel<D, CAP, BIAS, FIXED, MODE, kEmu>>((int)bytes)));
  US_CUDA_CHECK(us::launch_pdl(scored_flash_kernel<D, CAP, BIAS, FIXED, MODE, kEmu>, grid, dim3(kThreads), bytes, stream, q, k, v, a));
  return US_OK;
}
template <int D, int MODE>
int start_any(bool cap, dim3 grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ScoredArgs& a,
              cudaStream_t stream) {
  const bool bias = a.slopes != nullptr;
  if (!cap) return bias ? start<D, false, true, false, MODE>(grid, q, k, v, a, stream) : start<D, false, false, false, MODE>(grid, q, k, v, a, stream);
  // (FP16 weights need a maximum: they end at 2^16)
  if (small_cap(a) && !a.q_back) return bias ? start<D, true, true, true, MODE>(grid, q, k, v, a, stream) : start<D, true, false, true, MODE>(grid, q, k, v, a, stream);
  return bias ? start<D, true, true, false, MODE>(grid, q, k, v, a, stream) : start<D, true, false, false, MODE>(grid, q, k, v, a, stream);
}
template <int MODE>
int start_any(int D, bool cap, dim3 grid, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const ScoredArgs& a,
              cudaStream_t stream) {
  return D == 128 ? start_any<128, MODE>(cap, grid, q, k, v, a, stream) : start_any<64, MODE>(cap, grid, q, k, v, a, stream);
}

}  // namespace

namespace {
// A tile has the largest power of two of a key head's query heads that divides them, with 128 rows shared out among
// them.  Few new rows behind long histories fill tiles that way (11 requests of 9 rows and 64 heads over 4 behind 3,600
// keys: 221 us with one head a tile, 66 so; 8 of 75 rows and 32 heads: 172, 106), and fewer blocks hang over a diagonal
// or a document's ends (ragged batch: 214, 197; documents: 115, 111; 4096 rows: 141, 144).  Where a bias grows fast and
// keys follow a row, the warp's steepest head decides for all (4096 rows that see all: 268, 293).
int pack_of(int share, int max_q) {
  int pack = 0;
  while (pack < 7 && share % (2 << pack) == 0 && ((long long)max_q << (pack + 1)) <= 65535LL * 2 * kBM) ++pack;
  return pack;
}
}  // namespace

// Parts that the keys of a prompt call go in: as many as fill the GPU once where few rows would leave half of it idle, of
// four blocks or more (37 rows of 32 heads over 8,000 keys: 107 us in one part, 28 in 36; 200 rows over 16,000: 111, 42).
// Parts are joined by a launch of their own; see us_scored_flash for their places.
US_API int us_scored_flash_parts(int n, int max_q, int max_k, int Hq, int Hkv) {
  int sms = 0;
  if (n < 1 || max_q < 1 || Hkv < 1 || Hq < Hkv || us::sm_count(&sms) != cudaSuccess) return 1;
  const int pack = pack_of(Hq / Hkv, max_q), blocks = (max_k + kBN - 1) / kBN;
  const long long ctas = (long long)(Hq >> pack) * n * ((((long long)max_q << pack) + 2 * kBM - 1) / (2 * kBM));
  const int parts = (int)min((long long)(blocks / 4), sms / ctas);
  if (parts < 2) return 1;
  const int each = (blocks + parts - 1) / parts;
  return (blocks + each - 1) / each;
}

// q [Tq, Hq, D], k / v [Tk, Hkv, D], out [Tq, Hq, D], bf16 with row pitches; cu_q / cu_k [n + 1].  docs [Tk] with ranges
// (int32 [2 (Tk / 128 + n + 1)], written here), prefix [n], slopes [Hq]: or null.  cap 0, window 0: none.  fill: output rows of
// no sequence become zeros (some warps of the launch have time for n max_q of them).  parts > 1: part_o,
// part_ml [parts][n][max_q][Hq][D and 2] take the parts' results.
US_API int us_scored_flash(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, void* out,
                           long long ldo, const int* cu_q, const int* cu_k, int n, int Tq, int Tk, int Hq, int Hkv, int D,
                           int max_q, int max_k, float scale, float cap, const float* slopes, int causal, int window,
                           const int* docs, const int* prefix, void* ranges, int fill, int parts, float* part_o, float* part_ml, void* stream_) {
  US_REQUIRE(q && k && v && out && cu_q && cu_k && n >= 1 && n <= 65535 && Tq >= 1 && Tk >= 1 && max_q >= 1 && max_q <= 65535 * 2 * kBM && max_k >= 0);
  US_REQUIRE((D == 64 || D == 128) && Hkv >= 1 && Hq >= 1 && Hq <= 65535 && Hq % Hkv == 0 && window >= 0 && cap >= 0.f);
  US_REQUIRE(((ldq | ldk | ldv | ldo) % 8) == 0 && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16) == 0);
  US_REQUIRE(!docs || ranges);
  US_REQUIRE(max_k <= kMaxBlocks * kBN && parts >= 1 && (parts == 1 || (part_o && part_ml)));
  const int pack = pack_of(Hq / Hkv, max_q);
  CUtensorMap tmQ, tmK, tmV;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)Tq};
  const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)ldq * 2};
  const uint32_t box[3] = {64, 1u << pack, (uint32_t)kBM >> pack};
  int rc = us_tmap_encode(&tmQ, q, US_TMAP_BF16, 3, dims, strides, box, US_SWZ_128);
  if (!rc) rc = us_tmap_2d(&tmK, k, US_TMAP_BF16, (uint64_t)Tk, (uint64_t)Hkv * D, (uint64_t)ldk, kBN, 64, US_SWZ_128);
  if (!rc) rc = us_tmap_2d(&tmV, v, US_TMAP_BF16, (uint64_t)Tk, (uint64_t)Hkv * D, (uint64_t)ldv, kBN, 64, US_SWZ_128);
  if (rc) return rc;
  cudaStream_t stream = (cudaStream_t)stream_;
  ScoredArgs a = {};
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.out = (__nv_bfloat16*)out;
  a.ldo = ldo;
  a.Tq = Tq;
  a.Tk = Tk;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.causal = causal;
  a.pack = pack;
  a.n = n;
  a.max_q = max_q;
  a.max_k = max_k;
  a.fill = fill;
  // (a window of all keys that a sequence may have is none; rows stand before the first key too, and their positions less the
  // window have to be 32-bit numbers)
  a.window = window < kMaxBlocks * kBN ? window : kMaxBlocks * kBN;
  a.docs = docs;
  a.prefix = prefix;
  a.ranges = (const int2*)ranges;
  a.status = us_status_ptr();
  set_rules(a, scale, cap, slopes);
  if (docs && max_k > 0)
    US_CUDA_CHECK(us::launch_pdl(doc_ranges_kernel, dim3(((max_k + kBN - 1) / kBN + 3) / 4, n), dim3(128), 0, stream, docs, cu_k, Tk, (int2*)ranges));
  const unsigned tiles = (unsigned)((((long long)max_q << pack) + 2 * kBM - 1) / (2 * kBM));
  if (parts == 1) return start_any<0>(D, cap > 0.f, dim3(Hq >> pack, n, tiles), tmQ, tmK, tmV, a, stream);
  a.parts = parts;
  a.blocks_per_part = ((max_k + kBN - 1) / kBN + parts - 1) / parts;
  a.part_o = part_o;
  a.part_ml = part_ml;
  rc = start_any<2>(D, cap > 0.f, dim3((Hq >> pack) * parts, n, tiles), tmQ, tmK, tmV, a, stream);
  if (rc) return rc;
  const long long rows = (long long)n * max_q * Hq;
  US_REQUIRE(rows < (1LL << 31));
  US_CUDA_CHECK(us::launch_pdl(D == 128 ? join_parts_kernel<128> : join_parts_kernel<64>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, a));
  return US_OK;
}

// The part that the shared prefixes of a decode batch have in its attention (scored_decode.cu): rows
// [cu_rows[g], cu_rows[g + 1]) of q [B, Hq, D] against the first shared[g] keys behind row cu_rows[g]'s page list in
// k / v [pages, page, Hkv, D], or, with key_stride > 0, in rows g * key_stride .. of packed k / v [key_rows, Hkv, D]; with q_back and
// exps q, k and v are FP16 (us_quant_prefix).  Of a prefix the first most_shared keys are taken at most: those that the page
// lists, the packed rows and the parts have room for.
// part_o, part_ml: [groups][pairs][Hkv][parts][256][D and 2].
US_API int us_scored_prefix(const void* q, long long ldq, const void* k, long long pages, const void* v, long long page,
                            const float* q_back, const void* exps, int key_stride, int most_shared, const int* table, int max_pages, int key_rows, int B, const int* lens,
                            const int* cu_rows, const int* shared, int groups, int Hq, int Hkv, int D, int max_rows, float scale,
                            float cap, const float* slopes, float* part_o, float* part_ml, int pairs, int parts,
                            int blocks_per_part, void* stream_) {
  US_REQUIRE(q && k && v && lens && cu_rows && shared && part_o && part_ml && table && key_stride >= 0 && (!q_back || (exps && key_stride > 0)) && groups >= 1 && groups <= 65535 && B >= 1);
  US_REQUIRE((D == 64 || D == 128) && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= kBM && cap >= 0.f && max_rows >= 1);
  US_REQUIRE((ldq % 8) == 0 && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16) == 0 && pairs >= 1 && parts >= 1 &&
             blocks_per_part >= 1 && blocks_per_part <= kMaxBlocks && (long long)pairs * Hkv <= 65535);
  const int share = Hq / Hkv, per = kBM / share;
  US_REQUIRE((long long)pairs * 2 * per >= max_rows);
  US_REQUIRE(most_shared >= 0 && (long long)most_shared <= (long long)parts * blocks_per_part * kBN && (key_stride == 0 || most_shared <= key_stride) &&
             page >= 1 && (long long)most_shared <= (long long)max_pages * page);
  uint64_t rows = (uint64_t)key_rows;
  uint32_t box = kBN;
  if (key_stride == 0) {
    US_REQUIRE(pages >= 1 && page >= 8 && (kBN % page == 0 || page % kBN == 0) && pages * page <= 0x7fffff00LL && max_pages >= 1);
    rows = (uint64_t)(pages * page);
    box = (uint32_t)(page < kBN ? page : kBN);
  }
  US_REQUIRE(rows >= 1);
  CUtensorMap tmQ, tmK, tmV;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)B};
  const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)ldq * 2};
  const uint32_t qbox[3] = {64, (uint32_t)share, (uint32_t)per};
  const int type = q_back ? US_TMAP_F16 : US_TMAP_BF16;
  int rc = us_tmap_encode(&tmQ, q, type, 3, dims, strides, qbox, US_SWZ_128);
  if (!rc) rc = us_tmap_2d(&tmK, k, type, rows, (uint64_t)Hkv * D, (uint64_t)Hkv * D, box, 64, US_SWZ_128);
  if (!rc) rc = us_tmap_2d(&tmV, v, type, rows, (uint64_t)Hkv * D, (uint64_t)Hkv * D, box, 64, US_SWZ_128);
  if (rc) return rc;
  ScoredArgs a = {};
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.table = table;
  a.max_pages = max_pages;
  a.pages = (int)pages;
  a.page = (int)page;
  a.q_back = q_back;
  a.exps = (const int2*)exps;
  a.key_stride = key_stride;
  a.most_shared = most_shared;
  a.lens = lens;
  a.cu_rows = cu_rows;
  a.shared = shared;
  a.batch = B;
  a.pairs = pairs;
  a.parts = parts;
  a.blocks_per_part = blocks_per_part;
  a.part_o = part_o;
  a.part_ml = part_ml;
  a.status = us_status_ptr();
  set_rules(a, scale, cap, slopes);
  return start_any<1>(D, cap > 0.f, dim3(parts, pairs * Hkv, groups), tmQ, tmK, tmV, a, (cudaStream_t)stream_);
}
