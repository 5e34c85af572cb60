// Softmax attention of one new token a sequence over cache pages: scores capped by a tanh, biased by distance, cut
// below a first visible key or a window; pages of bf16, or of 8- or 4-bit integers (quant_pages.cu); batches whose
// sequences share a prefix, whose part of the result comes from scored_flash_tc05.cu.
//
//   s = scale q.k_j;  s = cap tanh(s / cap);  s -= slope_h (p - j), p = length - 1;  first <= j < length
//   out_h = sum_j e^s v_j / sum_j e^s                       (zeros where no key is visible)
//
// Bound by the bytes of the keys, so everything serves the stream of loads:
//
// * All keys of the launch form one list of tiles ordered by (sequence, key head, tile), cut into one range per SM:
//   no SM idles behind a long sequence.  A range that starts or ends inside a (sequence, key head) pair leaves that
//   pair's unnormalised output, maximum and sum in the CTA's slot (0: its first pair, 1: its last); the CTA whose
//   arrival completes a pair's count folds the slots and puts the count back to zero.
// * Each of eight warps has its own KW keys of every tile and its own ring of stages, which it fills itself
//   with 16-byte asynchronous copies: page ids of a tile are one load per lane, a tile ahead of its copies, and no
//   warp waits for another until a pair ends.  The ring runs on across pairs.
// * Keys stand on the M side of m16n8k16 products (S^T = K Q^T, O^T = V^T P^T), the query heads of a key head on the
//   N side: groups of up to 8 heads pay for 8 columns, not for 16 rows, and the softmax has its maximum and sum
//   per column, three shuffles each.  P^T becomes the B operand by an 8 x 8 transpose in registers (movmatrix).
// * Integer codes become bf16 exactly (8 bits: (0x4300 | low 7 bits) - (0x4300 | sign bit) = 128 + l - 128 (1 + sign);
//   4 bits: (0x4300 | u) - 136), three or two and a half instructions per two codes, and never carry a scale: a key's
//   scales multiply its scores, a value's its probabilities.  Which channel stands in which k slot is free as long as
//   Q agrees, so bytes and nibbles are taken out of the words as they lie; for V the free order is the order of the
//   output rows.
//
// Statistics and outputs are FP32; P (with a value's scale) is rounded to bf16 for its product, at most 2^-9 of each
// weight.  Keys that are not visible are never loaded (zeros in their place), so nothing in them reaches the result.
#include "include/us_common.cuh"
#include "include/us_mma.cuh"

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSeqs = 1024;
constexpr int kPitch = 68;                  // floats per head in the merge buffer: 8 rows x 4 heads on 32 banks

struct DecodeArgs {
  const __nv_bfloat16* q;
  const uint8_t *kc, *vc;
  const __nv_bfloat16 *ks, *vs;             // scales of integer pages
  const int *table, *lens, *starts;
  __nv_bfloat16* out;
  float *part_o, *part_ml;                  // [CTAs][2][16][D], [CTAs][2][16][2]
  int* counters;                            // [B * pairs per sequence], zero between launches
  const float* slopes;
  long long ldq, ldo;
  int B, Hq, Hkv, chunks, max_pages, pages, page, shift, window;
  float scale_log2, scale_cap, cap_log2;    // cap_log2 == 0: no cap; scale_cap = 2 scale log2(e) / cap
  // shared prefixes: rows [cu_rows[g], cu_rows[g + 1]) share their first shared[g] keys, whose partial results are
  // pre_o / pre_ml [group][tile pair][key head][part][256][D or 2]
  const int *cu_rows, *shared;
  const float *pre_o, *pre_ml;
  int groups, pairs, parts, blocks_per_part;
  unsigned int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // 8 x 8 matrix of 16-bit values across the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp16z(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4z(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bytes_even(uint32_t x) {   // bytes 0 and 2 as bf16
  return sub_bf2((x & 0x007f007fu) | 0x43004300u, (x & 0x00800080u) | 0x43004300u);
}
__device__ __forceinline__ uint32_t bytes_odd(uint32_t x) { return bytes_even(x >> 8); }
template <int N>
__device__ __forceinline__ uint32_t nibbles(uint32_t x) {      // nibbles N and N + 4 as bf16
  return sub_bf2(((x >> (4 * N)) & 0x000f000fu) | 0x43004300u, 0x43084308u);
}

// A position in the tile list.
struct Walk {
  int b, hc, t, tiles;
};

template <int D, int FMT>                   // FMT: bits of a code (16: bf16)
struct Shape {
  static constexpr int kRow = D * FMT / 8;                          // bytes of a cached row
  static constexpr int kKeys = kRow >= 256 ? 16 : 32;               // keys of a warp's stage
  static constexpr int kScales = FMT == 16 ? 0 : kKeys * 4;         // bytes of a plane's scales
  static constexpr int kStage = 2 * kKeys * kRow + 2 * kScales;
  static constexpr int kRoom = 196608 / kWarps;                     // ring bytes of a warp
  static constexpr int kStages = kRoom / kStage > 6 ? 6 : kRoom / kStage;
  static constexpr int kTile = kWarps * kKeys;
  static constexpr int kPieces = kRow / 16;                         // 16-byte pieces of a row
};

template <int PIECES>
__device__ __forceinline__ int swizzle(int row, int piece) {        // eight rows' same piece: eight bank groups
  if constexpr (PIECES >= 8) return piece ^ (row & 7);
  else if constexpr (PIECES == 4) return piece ^ ((row >> 1) & 3);
  else return piece ^ ((row >> 2) & 1);
}

constexpr int kMergeFloats = kWarps * 8 * kPitch;                   // [warp][8 heads][64 channels + 4]

template <int D, int FMT>
constexpr size_t shared_bytes() {
  using S = Shape<D, FMT>;
  return (size_t)kWarps * S::kStages * S::kStage + kMergeFloats * 4 + (kWarps * 32 + 32) * 4 + (3 * kMaxSeqs + 4) * 4;
}

template <int D, int FMT, int NT>           // NT: 8-column head tiles (query heads of a key head in one pass: 8 NT)
__global__ void __launch_bounds__(kThreads, 1) scored_decode_kernel(const DecodeArgs a) {
  using S = Shape<D, FMT>;
  constexpr int KW = S::kKeys, MT = KW / 16, KS = D / 16, G = D / 64;
  US_PDL_PROLOGUE();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem + (size_t)warp * S::kStages * S::kStage;
  float* buf = (float*)(smem + (size_t)kWarps * S::kStages * S::kStage);
  float* ml = buf + kMergeFloats;           // [warp][16 heads][2]
  int* flag = (int*)(ml + kWarps * 32);     // [0]: this CTA completes the pair
  int* pre = flag + 32;                     // tiles before sequence b
  int* first = pre + kMaxSeqs + 4;          // visible keys of sequence b: [first, end)
  int* end = first + kMaxSeqs;

  // ---- the tile list ----
  const int B = a.B, Hc = a.Hkv * a.chunks;
  for (int b = tid; b < B; b += kThreads) {
    int len = max(a.lens[b], 0), lo = a.starts ? max(a.starts[b], 0) : 0;
    if (a.window > 0) lo = max(lo, len - a.window);
    if (a.groups > 0) {
      int g = 0, h = a.groups - 1;
      while (g < h) {
        const int mid = (g + h + 1) >> 1;
        if (a.cu_rows[mid] <= b) g = mid; else h = mid - 1;
      }
      if (b < a.cu_rows[a.groups]) lo = max(lo, a.shared[g]);
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
    pre[b + 1] = max(1, (hi - lo + S::kTile - 1) / S::kTile);       // a pair without keys still has its zeros to write
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
  const int n_cta = min((int)gridDim.x, total), cta = blockIdx.x;
  if (cta >= n_cta) return;
  auto range = [&](int c) { return (int)(((long long)c * total) / n_cta); };
  auto owner = [&](int g) {
    int c = (int)(((long long)g * n_cta) / total);
    while (c + 1 < n_cta && range(c + 1) <= g) ++c;
    while (c > 0 && range(c) > g) --c;
    return c;
  };
  const int g0 = range(cta), g1 = range(cta + 1);
  Walk load;
  {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (Hc * pre[mid] <= g0) lo = mid; else hi = mid - 1;
    }
    load.b = lo;
    load.tiles = pre[lo + 1] - pre[lo];
    const int r = g0 - Hc * pre[lo];
    load.hc = r / load.tiles;
    load.t = r - load.hc * load.tiles;
  }
  Walk cur = load;
  auto advance = [&](Walk& w) {
    if (++w.t < w.tiles) return;
    w.t = 0;
    if (++w.hc < Hc) return;
    w.hc = 0;
    ++w.b;
    if (w.b < B) w.tiles = pre[w.b + 1] - pre[w.b];
  };

  // ---- loads: this warp's keys of a tile into one of its stages ----
  // the slot (page * page size + offset) of lane's key in the tile at w, -1 where there is none
  auto slot_of = [&](const Walk& w) -> int {
    const int j = first[w.b] + w.t * S::kTile + warp * KW + lane;
    if (lane >= KW || j >= end[w.b]) return -1;
    const int pi = a.shift >= 0 ? j >> a.shift : j / a.page;
    const int pg = __ldg(a.table + (long long)w.b * a.max_pages + pi);
    if ((unsigned)pg >= (unsigned)a.pages) {
      us_dev_fail(a.status, US_DEV_BOUNDS);
      return -1;
    }
    return pg * a.page + (j - pi * a.page);
  };
  int loaded = g0;                          // tiles up to here have been asked for
  int slot_next = slot_of(load);
  auto issue = [&](int stage) {
    if (loaded < g1) {
      const int slot = slot_next, hk = load.hc / a.chunks;
      uint8_t* st = ring + stage * S::kStage;
      const uint32_t kd = (uint32_t)__cvta_generic_to_shared(st), vd = kd + KW * S::kRow;
      constexpr int kRows = 32 / S::kPieces;       // rows that one instruction of the warp brings
      const int piece = lane % S::kPieces;
#pragma unroll
      for (int i = 0; i < KW / kRows; ++i) {
        const int r = i * kRows + lane / S::kPieces;
        const int sl = __shfl_sync(0xffffffffu, slot, r);
        const long long off = sl < 0 ? 0 : ((long long)sl * a.Hkv + hk) * S::kRow + piece * 16;
        const uint32_t to = r * S::kRow + swizzle<S::kPieces>(r, piece) * 16;
        cp16z(kd + to, a.kc + off, sl >= 0);
        cp16z(vd + to, a.vc + off, sl >= 0);
      }
      if constexpr (FMT != 16) {            // 4 bytes of scales a key: two groups, or one beside its neighbour's
        if (lane < KW) {
          const int pg = slot < 0 ? 0 : a.shift >= 0 ? slot >> a.shift : slot / a.page;
          const long long at = (((long long)pg * a.Hkv + hk) * a.page + (slot < 0 ? 0 : slot - pg * a.page)) * G;
          const uint32_t sd = kd + 2 * KW * S::kRow + lane * 4;
          cp4z(sd, a.ks + (at & ~1LL), slot >= 0);
          cp4z(sd + KW * 4, a.vs + (at & ~1LL), slot >= 0);
        }
      }
      ++loaded;
      if (loaded < g1) {
        advance(load);
        slot_next = slot_of(load);
      }
    }
    us::cp_commit();
  };

  const int c4 = lane & 3, r8 = lane >> 2;
  uint32_t qf[NT][KS][2];
  float m[NT][2], l[NT][2], bias[NT][2], o[KS][NT][4];
  auto begin_pair = [&]() {
    const int hk = cur.hc / a.chunks, chunk = cur.hc - hk * a.chunks;
    const int share = a.Hq / a.Hkv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int gi = chunk * 16 + nt * 8 + r8;
      const __nv_bfloat16* row = a.q + (long long)cur.b * a.ldq + (long long)(hk * share + gi) * D;
      const bool there = gi < share;
#pragma unroll
      for (int k = 0; k < KS; ++k) qf[nt][k][0] = qf[nt][k][1] = 0;
      if (there) {
        if constexpr (FMT == 16) {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            qf[nt][k][0] = *reinterpret_cast<const uint32_t*>(row + k * 16 + c4 * 2);
            qf[nt][k][1] = *reinterpret_cast<const uint32_t*>(row + k * 16 + c4 * 2 + 8);
          }
        } else if constexpr (FMT == 8) {
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
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = chunk * 16 + nt * 8 + c4 * 2 + e;
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
        bias[nt][e] = a.slopes && h < share ? a.slopes[hk * share + h] * 1.4426950408889634f : 0.f;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
    }
  };

  // ---- one stage: S^T = K Q^T, the softmax's step, O^T += V^T P^T ----
  auto consume = [&](int stage) {
    const int j0 = first[cur.b] + cur.t * S::kTile + warp * KW, hi = end[cur.b];
    if (j0 >= hi) return;
    const uint8_t* st = ring + stage * S::kStage;
    const uint32_t kd = (uint32_t)__cvta_generic_to_shared(st), vd = kd + KW * S::kRow;
    const uint32_t* sk = reinterpret_cast<const uint32_t*>(st + 2 * KW * S::kRow);
    const uint32_t* sv = sk + KW;
    // a key's two scales (64 channels: its one, which is the half that its parity says, the page size being even)
    auto scales = [&](const uint32_t* s, int key, float (&f)[G]) {
      const uint32_t w = s[key];
      if constexpr (G == 2) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
      } else {
        f[0] = __uint_as_float((j0 + key) & 1 ? w & 0xffff0000u : w << 16);
      }
    };
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float acc[G][NT][4];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[g][nt][e] = 0.f;
      const int row = mt * 16 + (lane & 15);
      if constexpr (FMT == 16) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t f[4];
          us::ldsm4(f, kd + row * S::kRow + swizzle<S::kPieces>(row, 2 * k + (lane >> 4)) * 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            us::mma16816(acc[0][nt], f[0], f[1], f[2], f[3], qf[nt][k][0], qf[nt][k][1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kPieces / 2; ++i) {
          uint32_t f[4];
          us::ldsm4(f, kd + row * S::kRow + swizzle<S::kPieces>(row, 2 * i + (lane >> 4)) * 16);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = f[2 * half], y = f[2 * half + 1];   // keys 0 - 7 and 8 - 15
            const int piece = 2 * i + half;
            if constexpr (FMT == 8) {
              const uint32_t a0 = bytes_even(x), a1 = bytes_even(y), a2 = bytes_odd(x), a3 = bytes_odd(y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                us::mma16816(acc[piece / 4][nt], a0, a1, a2, a3, qf[nt][piece][0], qf[nt][piece][1]);
            } else {
              const uint32_t a0 = nibbles<0>(x), a1 = nibbles<0>(y), a2 = nibbles<1>(x), a3 = nibbles<1>(y);
              const uint32_t b0 = nibbles<2>(x), b1 = nibbles<2>(y), b2 = nibbles<3>(x), b3 = nibbles<3>(y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                us::mma16816(acc[piece / 2][nt], a0, a1, a2, a3, qf[nt][2 * piece][0], qf[nt][2 * piece][1]);
                us::mma16816(acc[piece / 2][nt], b0, b1, b2, b3, qf[nt][2 * piece + 1][0], qf[nt][2 * piece + 1][1]);
              }
            }
          }
        }
      }
      if constexpr (FMT == 16) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][nt][e] = acc[0][nt][e];
      } else {
        float f0[G], f1[G];
        scales(sk, mt * 16 + r8, f0);
        scales(sk, mt * 16 + r8 + 8, f1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = acc[0][nt][e] * (e < 2 ? f0[0] : f1[0]);
            if constexpr (G == 2) x = fmaf(acc[1][nt][e], e < 2 ? f0[1] : f1[1], x);
            s[mt][nt][e] = x;
          }
      }
    }
    // scores in units of log2(e)
    const int away0 = a.lens[cur.b] - 1 - j0;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = mt * 16 + r8 + (e >> 1) * 8;
          float x = s[mt][nt][e];
          if (a.cap_log2 > 0.f) {           // tanh y = 1 - 2 / (1 + e^(2 y)): off by some 2^-23 of the cap
            x = fmaf(-2.f * a.cap_log2, __frcp_rn(1.f + ex2(x * a.scale_cap)), a.cap_log2);
          } else {
            x *= a.scale_log2;
          }
          x = fmaf(-bias[nt][e & 1], (float)(away0 - key), x);
          if (j0 + key >= hi) x = -INFINITY;
          s[mt][nt][e] = x;
          top[nt][e & 1] = fmaxf(top[nt][e & 1], x);
        }
    }
    bool grown = false;
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = top[nt][e];
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        t = fmaxf(t, m[nt][e]);
        alpha[nt][e] = t == -INFINITY ? 1.f : ex2(m[nt][e] - t);
        grown |= t > m[nt][e];
        m[nt][e] = t;
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        l[nt][0] *= alpha[nt][0];
        l[nt][1] *= alpha[nt][1];
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nt][e] *= alpha[nt][e & 1];
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t pb[G][NT][2];
      float f0[G], f1[G];
      if constexpr (FMT != 16) {
        scales(sv, mt * 16 + r8, f0);
        scales(sv, mt * 16 + r8 + 8, f1);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[mt][nt][e];
          p[e] = x == -INFINITY ? 0.f : ex2(x - m[nt][e & 1]);
          l[nt][e & 1] += p[e];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (FMT == 16) {
            if (g == 0) {
              pb[0][nt][0] = transposed(us::pack_bf(p[0], p[1]));
              pb[0][nt][1] = transposed(us::pack_bf(p[2], p[3]));
            }
          } else {
            pb[g][nt][0] = transposed(us::pack_bf(p[0] * f0[g], p[1] * f0[g]));
            pb[g][nt][1] = transposed(us::pack_bf(p[2] * f1[g], p[3] * f1[g]));
          }
        }
      }
      if constexpr (FMT == 16) {
        const int row = mt * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t f[4];
          us::ldsm4t(f, vd + row * S::kRow + swizzle<S::kPieces>(row, 2 * i + ((lane >> 3) & 1)) * 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            us::mma16816(o[i][nt], f[0], f[1], f[2], f[3], pb[0][nt][0], pb[0][nt][1]);
        }
      } else {
        const int row = mt * 16 + (lane & 15);
#pragma unroll
        for (int i = 0; i < S::kPieces / 2; ++i) {
          uint32_t f[4];
          us::ldsm4t(f, vd + row * S::kRow + swizzle<S::kPieces>(row, 2 * i + (lane >> 4)) * 16);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = f[2 * half], y = f[2 * half + 1];   // keys 0 - 7 and 8 - 15
            const int piece = 2 * i + half;
            if constexpr (FMT == 8) {
              const uint32_t a0 = bytes_even(x), a1 = bytes_odd(x), a2 = bytes_even(y), a3 = bytes_odd(y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                us::mma16816(o[piece][nt], a0, a1, a2, a3, pb[piece / 4][nt][0], pb[piece / 4][nt][1]);
            } else {
              const uint32_t a0 = nibbles<0>(x), a1 = nibbles<1>(x), a2 = nibbles<0>(y), a3 = nibbles<1>(y);
              const uint32_t b0 = nibbles<2>(x), b1 = nibbles<3>(x), b2 = nibbles<2>(y), b3 = nibbles<3>(y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                us::mma16816(o[2 * piece][nt], a0, a1, a2, a3, pb[piece / 2][nt][0], pb[piece / 2][nt][1]);
                us::mma16816(o[2 * piece + 1][nt], b0, b1, b2, b3, pb[piece / 2][nt][0], pb[piece / 2][nt][1]);
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

  // folds the partial results of head `gi` of pair (b, hc), channels d and d + 1, that other launches and CTAs left:
  // slots of CTAs [c0, c1] and the parts of the shared prefix, beside (M, L, x, y)
  auto fold = [&](int b, int hc, int gi, int d, int c0, int c1, int begin, float M, float L, float x, float y) {
    const int hk = hc / a.chunks, chunk = hc - hk * a.chunks, share = a.Hq / a.Hkv;
    int np = 0;
    long long at = 0;
    if (a.groups > 0 && b < a.cu_rows[a.groups]) {
      int g = 0, h = a.groups - 1;
      while (g < h) {
        const int mid = (g + h + 1) >> 1;
        if (a.cu_rows[mid] <= b) g = mid; else h = mid - 1;
      }
      const int blocks = (a.shared[g] + 127) >> 7;
      np = min((blocks + a.blocks_per_part - 1) / a.blocks_per_part, a.parts);
      const int per = 128 / share, r = b - a.cu_rows[g];       // sequences of a 128-row tile of the prefix kernel
      if (blocks > a.parts * a.blocks_per_part || r >= a.pairs * 2 * per) {   // a group larger than the host was told
        us_dev_fail(a.status, US_DEV_BOUNDS);
        if (r >= a.pairs * 2 * per) np = 0;
      }
      const int tile = r / per, in_tile = (r - tile * per) * share + chunk * 16 + gi;
      at = ((((long long)g * a.pairs + (tile >> 1)) * a.Hkv + hk) * a.parts) * 256 + (tile & 1) * 128 + in_tile;
    }
    auto slot = [&](int c) { return ((long long)c * 2 + (range(c) >= begin ? 0 : 1)) * 16 + gi; };
    float top = M;
    for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(a.part_ml + slot(c) * 2));
    for (int i = 0; i < np; ++i) top = fmaxf(top, __ldcg(a.pre_ml + (at + (long long)i * 256) * 2));
    float w = M == -INFINITY ? 0.f : ex2(M - top);
    L *= w;
    x *= w;
    y *= w;
    auto add = [&](const float* mls, const float* os) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(mls));
      const float u = v.x == -INFINITY ? 0.f : ex2(v.x - top);
      const float2 p = __ldcg(reinterpret_cast<const float2*>(os));
      L = fmaf(u, v.y, L);
      if (u != 0.f) {          // a part of weight zero may hold anything
        x = fmaf(u, p.x, x);
        y = fmaf(u, p.y, y);
      }
    };
    for (int c = c0; c <= c1; ++c) add(a.part_ml + slot(c) * 2, a.part_o + slot(c) * D + d);
    for (int i = 0; i < np; ++i) add(a.pre_ml + (at + (long long)i * 256) * 2, a.pre_o + (at + (long long)i * 256) * D + d);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint32_t*>(a.out + (long long)b * a.ldo + (long long)(hk * share + chunk * 16 + gi) * D + d) =
        us::pack_bf(x * inv, y * inv);
  };

#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);
  int stage = 0, segment = 0, i = g0;
  while (i < g1) {
    begin_pair();
    const int n = min(cur.tiles - cur.t, g1 - i);
    const bool whole = cur.t == 0 && n == cur.tiles;
    for (int t = 0; t < n; ++t, ++i, ++cur.t) {
      us::cp_wait<S::kStages - 2>();
      __syncwarp();
      consume(stage);
      __syncwarp();
      issue(stage == 0 ? S::kStages - 1 : stage - 1);    // the stage that the tile before this one has left
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }
    // ---- the pair (or this CTA's part of it) ends: the warps' results become one ----
    const int hk = cur.hc / a.chunks, chunk = cur.hc - hk * a.chunks, share = a.Hq / a.Hkv;
    const int heads = min(8 * NT, share - chunk * 16);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = l[nt][e];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        if (r8 == 0) {
          const int h = nt * 8 + c4 * 2 + e;
          ml[(warp * 16 + h) * 2] = m[nt][e];
          ml[(warp * 16 + h) * 2 + 1] = t;
        }
      }
    __syncthreads();
    const long long slot0 = ((long long)cta * 2 + (segment == 0 ? 0 : 1)) * 16;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = nt * 8 + c4 * 2 + e;
        float top = ml[h * 2];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, ml[(k * 16 + h) * 2]);
        w[e] = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - top);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {          // 64 channels of eight heads at a time
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const int t = g * 4 + i4;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            buf[(warp * 8 + c4 * 2 + (e & 1)) * kPitch + channel(t, e >> 1) - g * 64] = w[e & 1] == 0.f ? 0.f : o[t][nt][e] * w[e & 1];
        }
        __syncthreads();
        const int h8 = tid >> 5, d = (tid & 31) * 2, h = nt * 8 + h8;
        if (h < heads) {
          float top = ml[h * 2];
#pragma unroll
          for (int k = 1; k < kWarps; ++k) top = fmaxf(top, ml[(k * 16 + h) * 2]);
          float x = 0.f, y = 0.f, L = 0.f;
#pragma unroll
          for (int k = 0; k < kWarps; ++k) {
            const float2 v = *reinterpret_cast<const float2*>(buf + (k * 8 + h8) * kPitch + d);
            x += v.x;
            y += v.y;
            const float mk = ml[(k * 16 + h) * 2];
            L += mk == -INFINITY ? 0.f : ml[(k * 16 + h) * 2 + 1] * ex2(mk - top);
          }
          if (whole) {
            fold(cur.b, cur.hc, h, g * 64 + d, 1, 0, 0, top, L, x, y);
          } else {
            *reinterpret_cast<float2*>(a.part_o + (slot0 + h) * D + g * 64 + d) = make_float2(x, y);
            if (g == 0 && (tid & 31) == 0)
              *reinterpret_cast<float2*>(a.part_ml + (slot0 + h) * 2) = make_float2(top, L);
          }
        }
        __syncthreads();
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      const int begin = Hc * pre[cur.b] + cur.hc * cur.tiles;
      const int c0 = owner(begin), c1 = owner(begin + cur.tiles - 1);
      if (tid == 0) {
        int* count = a.counters + cur.b * Hc + cur.hc;
        const int last = atomicAdd(count, 1) == c1 - c0;
        if (last) *count = 0;
        flag[0] = last;
      }
      __syncthreads();
      if (flag[0]) {
        __threadfence();
        for (int e = tid; e < heads * (D / 2); e += kThreads)
          fold(cur.b, cur.hc, e / (D / 2), (e % (D / 2)) * 2, c0, c1, begin, -INFINITY, 0.f, 0.f, 0.f);
      }
      __syncthreads();
    }
    ++segment;
    --cur.t;                                 // the loop above left it one past the pair's last tile
    advance(cur);
  }
}

template <int D, int FMT, int NT>
int launch(const DecodeArgs& a, int ctas, cudaStream_t stream) {
  const size_t bytes = shared_bytes<D, FMT>();
  static_assert(shared_bytes<D, FMT>() <= 232448, "shared memory");
  US_CUDA_CHECK((us::allow_shared<scored_decode_kernel<D, FMT, NT>>((int)bytes)));
  US_CUDA_CHECK(us::launch_pdl(scored_decode_kernel<D, FMT, NT>, dim3(ctas), dim3(kThreads), bytes, stream, a));
  return US_OK;
}

}  // namespace

// Bytes of the partial results of a launch on the current device (its counters: B * Hkv * ceil(Hq / Hkv / 16) int32).
US_API long long us_scored_decode_scratch(int D) {
  int sms = 0;
  if (us::sm_count(&sms) != cudaSuccess) return -1;
  return (long long)sms * 2 * 16 * (D + 2) * (long long)sizeof(float);
}

// q [B, Hq, D] bf16 (row pitch ldq); pages [pages, page, Hkv, D] bf16 or integer codes with scales (bits 8, 4; 16: bf16);
// table [B, max_pages], lens [B], starts [B] or null.  scratch, counters: see above; counters are zero before the first
// call and left zero; calls that share them are ordered on the device.  groups > 0: the keys below shared[g] of rows
// [cu_rows[g], cu_rows[g + 1]) are in pre_o / pre_ml (us_scored_flash), whose layout the last arguments give.
US_API int us_scored_decode(const void* q, long long ldq, const void* kc, const void* vc, const void* ks, const void* vs,
                            const int* table, int max_pages, const int* lens, const int* starts, void* out, long long ldo,
                            void* scratch, int* counters, int B, int Hq, int Hkv, int D, int bits, int pages, int page,
                            int window, float scale, float cap, const float* slopes, int groups, const int* cu_rows,
                            const int* shared, const float* pre_o, const float* pre_ml, int pairs, int parts,
                            int blocks_per_part, void* stream_) {
  US_REQUIRE(B >= 0 && B <= kMaxSeqs && (D == 64 || D == 128) && Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0);
  if (B == 0) return US_OK;
  US_REQUIRE(q && kc && vc && table && lens && out && scratch && counters && max_pages >= 1 && pages >= 1 && page >= 1);
  US_REQUIRE(bits == 16 || ((bits == 8 || bits == 4) && ks && vs && page % 2 == 0 && (((uintptr_t)ks | (uintptr_t)vs) % 4) == 0));
  US_REQUIRE((long long)pages * page <= 0x7fffffffLL && window >= 0 && cap >= 0.f);
  US_REQUIRE((ldq % 8) == 0 && (ldo % 2) == 0 && (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) % 16) == 0 &&
             ((uintptr_t)out % 4) == 0);
  const int share = Hq / Hkv;
  if (groups > 0) US_REQUIRE(cu_rows && shared && pre_o && pre_ml && pairs >= 1 && parts >= 1 && blocks_per_part >= 1 && share <= 128 &&
                             window == 0 && !starts);
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
  a.part_o = (float*)scratch;
  a.part_ml = (float*)scratch + (long long)sms * 2 * 16 * D;
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
  a.cu_rows = cu_rows;
  a.shared = shared;
  a.pre_o = pre_o;
  a.pre_ml = pre_ml;
  a.pairs = pairs;
  a.parts = parts;
  a.blocks_per_part = blocks_per_part;
  a.status = us_status_ptr();
  cudaStream_t stream = (cudaStream_t)stream_;
#define US_SCORED(DD, F)                                                                   \
  if (D == DD && bits == F) return share <= 8 ? launch<DD, F, 1>(a, sms, stream) : launch<DD, F, 2>(a, sms, stream)
  US_SCORED(64, 16);
  US_SCORED(64, 8);
  US_SCORED(64, 4);
  US_SCORED(128, 16);
  US_SCORED(128, 8);
  US_SCORED(128, 4);
#undef US_SCORED
  return US_ERR_UNSUPPORTED;
}
