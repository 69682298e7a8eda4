// Attention over paged 4-bit K/V (nsa_kv4.h) on gfx950, up to three sources with their gated mix.
//
// For query row i of request b at position p, per source s over the visible keys j:
//   o_s = sum_j exp(scale q k_j - m) v_j / sum_j exp(scale q k_j - m),   out = sum_s gate_s o_s.
// A workgroup takes up to 16 heads of a KV group at one query row, its waves 32 keys at a time with a
// running maximum and sum.  Rows of moderate length are one workgroup's whole work (kv4_split: when).
// Otherwise the keys of each source are cut into parts, a workgroup a part, which writes one partial
// {max, sum, O} to the workspace; a second kernel joins the parts of each head.  The number of
// parts is the host's (lengths are on the device, so it goes by what they may be), the same for every
// request; how many keys a part holds follows on the device from the request's own count, so that a short
// request uses few parts.  A request much longer than the rest of its batch has no more of them
// than they may have (kv4_split: what that costs).
//
// Bound, 131072 keys of H64 G4 dk 192 dv 128 (91 MB): memory while it runs, 98 MB of L2 misses in the 16 us
// that its waves live (6.1 TB/s; the vector units are busy 42 % of that time, a wave waits for 50 %), within
// a launch of 20 us, and 6 us for the join.  Small calls are bound by latency: a launch
// of 2 us, then arguments -> length -> table -> rows one behind the other.
//
// Per wave and tile: S^T = K Q^T with K from the page: lane (g, r) reads the quarter g of key r's
// row, D / 8 bytes, which is its share of every product step (the k slots of a step may stand for any
// features as long as Q's agree), turned into bf16 in registers.  V rows go through LDS as bf16 and
// come back transposed.  Queries and probabilities in fp32 are split into three bf16 parts that hold
// all 24 bits (x = hi + mid + lo, each the rounding of what is left): the cached values are exact in
// bf16, so three bf16 products replace each fp32 one, at the accuracy of fp32.  With bf16 queries each
// probability is rounded to bf16 for the second product (by 2^-8 of it at most; their sum is of the unrounded
// ones, in fp32), as in the other attention kernels here: one product instead of two.  Over values of any
// sign that adds about what rounding the output does: 2.0e-3 to 2.3e-3 from the 64-bit result (norm of the
// difference over its norm), where that result rounded to bf16 is 1.65e-3 from it.
#include <float.h>
#include <limits.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/nsa_hip.h"
#include "nsa_kv4.h"

namespace nsa {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kKvTile = 32, kKvWaves = 4;
constexpr int kKvStep = kKvTile * kKvWaves;  // keys of one round of a workgroup

struct Kv4Source {
  Kv4Pages pg;
  const int* tables;
  int64_t st_b;
  int W, cap;  // table entries, tokens they stand for
  IntDiv parts;
};

struct Kv4Attn {
  const void* q;
  int64_t sq_b, sq_h, sq_t;
  void* out;
  int64_t so_b, so_h, so_t;
  const void* gates;
  int64_t sg_b, sg_h, sg_t, sg_k;
  const int64_t* idx;  // [B][G][Tq][nslots]
  const int* lengths;
  Kv4Source src[3];
  float *part_ml, *part_o;  // workspace, per part and head of a tile: {max, sum}; then O [16][DV]
  IntDiv groups, tiles, blocks, d;  // by G, head tiles, lprime and d
  IntDiv heads, rows, hpgd;         // by H, Tq and hpg
  int n_rows;                       // B Tq H
  int parts[3];                     // of each source (0: absent)
  int whole;                        // a workgroup a query row tile, without parts
  int nparts, B, G, hpg, Tq, l, nslots, lprime, window, act;
  float scale;
};

// The arguments come from memory as well, and the compiler asks for each where it is first used, one
// latency after another.  Pinned scalars are asked for together.
template <typename T>
__device__ __forceinline__ void pin_one(T x) {
  asm volatile("" ::"s"(x));
}
template <typename... Ts>
__device__ __forceinline__ void pin(Ts... x) {
  (pin_one(x), ...);
}

// A wave-uniform element of memory that no kernel in flight writes, through the scalar cache.
__device__ __forceinline__ int scalar_load(const int* p, int i) {
  return reinterpret_cast<const int __attribute__((address_space(4)))*>(reinterpret_cast<uintptr_t>(p))[i];
}

// A wave's base address in memory and the load of a lane's element at a byte offset from it.
typedef const uint8_t __attribute__((address_space(1)))* wave_ptr;
__device__ __forceinline__ wave_ptr wave_base(const uint8_t* p, int64_t off) {
  uint64_t x = reinterpret_cast<uint64_t>(p) + off;
  asm volatile("" : "+s"(x));
  return reinterpret_cast<wave_ptr>(x);
}
template <typename V>
__device__ __forceinline__ V load_at(wave_ptr p, uint32_t off) {
  return *reinterpret_cast<const V __attribute__((address_space(1)))*>(p + off);
}

// What the keys of a query row follow from.
struct Kv4Shape {
  int l, nslots, lprime, window;
  IntDiv d;
};
// Entries of source s's key list for a query at position p (none for p < 0) and the first key of the
// list (the window's starts at a multiple of 16, masked below its real start); a list ends where
// the table, of cap tokens, does.
__device__ __forceinline__ int kv4_keys(const Kv4Shape& a, int s, int cap, int p, int* base) {
  const int n = p + 1, from = (n - min(a.window, n)) & ~15;
  const int cmp = n >= a.l ? min(cap, a.d.div(n - a.l) + 1) : 0;
  const int win = max(min(cap, n) - from, 0);
  *base = s == kDecWin ? from : 0;
  return p < 0 ? 0 : s == kDecSel ? a.nslots * a.lprime : s == kDecCmp ? cmp : win;
}
// keys of each of the source's parts (a multiple of a round)
__device__ __forceinline__ int kv4_part_keys(int keys, IntDiv parts) {
  const int each = parts.div(keys + parts.d - 1);  // keys at most 2^30
  return (each + kKvStep - 1) / kKvStep * kKvStep;
}

// x = sum of NS bf16 parts, each the rounding of what the ones before leave
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t* w) {
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    w[n] = pack_bf16x2(x, y);
    if (n + 1 < NS) {
      x -= __uint_as_float(w[n] << 16);
      y -= __uint_as_float(w[n] & 0xffff0000u);
    }
  }
}

// 4-bit rows of a wave's 32 keys on their way: the lane's quarter of keys c16 and 16 + c16, its
// 16-byte blocks of V rows, and their scales.
template <int DK, int DV>
struct Kv4Tile {
  static constexpr int NJ = DK / 32;  // words of a quarter row = product steps
  static constexpr int LPR = DV / 32, NV = (kKvTile * LPR + 63) / 64;  // lanes (16-byte blocks) of a V row, loads of a tile
  uint32_t k[2][NJ], ks[2][DK == 192 ? 2 : 1];
  uint4 v[NV];
  uint32_t vs[NV];
};

// word j of a quarter row's scale: a block of 32 features is four words, and a quarter of 192 features
// (48) starts or ends in the middle of one
template <int DK>
__device__ __forceinline__ uint32_t kv4_scale(uint32_t lo, uint32_t hi, int j, int g4) {
  if constexpr (DK != 192) return lo;
  else return j < 2 ? lo : j >= 4 ? hi : g4 & 1 ? hi : lo;
}

// The gate of source s from a row's three gate inputs.
__device__ __forceinline__ float kv4_gate(int act, int s, float z0, float z1, float z2) {
  const float z = s == 0 ? z0 : s == 1 ? z1 : z2;
  if (act == 1) return 1.f / (1.f + expf(-z));
  if (act == 2) {
    const float m = fmaxf(z0, fmaxf(z1, z2));
    return expf(z - m) / (expf(z0 - m) + expf(z1 - m) + expf(z2 - m));
  }
  return z;
}

// waves a SIMD that a kernel's registers leave room for, and waves of a workgroup that takes a row's
// whole work: as many as its registers and LDS allow on a CU.  Held to that, some put bytes of a lane into
// scratch: bf16 dk 192 12 (two registers; whole) and 48, fp32 dk 192 48 (whole) and 64, fp32 dk 128 48 (parts)
__host__ __device__ constexpr int kv4_waves(int esz, int dk) { return esz == 2 ? 4 : dk == 192 ? 2 : dk == 128 ? 3 : 4; }
__host__ __device__ constexpr int kv4_whole_waves(int esz, int dk) { return esz == 2 || dk <= 64 ? 16 : 8; }

// WHOLE: one workgroup of NW waves takes every key of every source of its query rows, the waves
// shared out among the sources by their tiles, and writes out itself: no partials and no second
// launch.  Otherwise one part of one source, of kKvWaves waves.
template <typename T, int DK, int DV, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(WHOLE ? NW / 4 : kv4_waves(sizeof(typename Store<T>::type), DK)))) void kv4_attn_kernel(Kv4Attn a) {
  using S = typename Store<T>::type;
  using Tile = Kv4Tile<DK, DV>;
  constexpr int NS = sizeof(S) == 2 ? 1 : 3;  // bf16 parts of a query or probability
  constexpr int NJ = Tile::NJ, LPR = Tile::LPR, NV = Tile::NV;
  constexpr int VP = DV + 16;  // staged V row pitch: row + 32 bytes, conflict-free transpose reads
  constexpr int VBYTES = NW * kKvTile * VP * 2;
  constexpr int OP = DV + 4, OBYTES = NW * 16 * OP * 4;  // row pitch of a wave's O: 16 lanes' rows in other banks
  static_assert(16 * (DK * sizeof(S) + 16) <= VBYTES, "the queries fit where V's rows go");
  __shared__ __attribute__((aligned(16))) char s_buf[VBYTES > OBYTES ? VBYTES : OBYTES];
  __shared__ float s_m[NW][16], s_l[NW][16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = lane >> 4, c16 = lane & 15;
  const IntDiv groups = a.groups, tiles = a.tiles;
  const Kv4Shape shape{a.l, a.nslots, a.lprime, a.window, a.d};
  const void* q = a.q;
  const int64_t sq_b = a.sq_b, sq_h = a.sq_h, sq_t = a.sq_t;
  const int64_t* idx = a.idx;
  const int* lengths = a.lengths;
  const int parts0 = a.parts[0], parts1 = a.parts[1], nparts = a.nparts, hpg = a.hpg, Tq = a.Tq;
  const float scale = a.scale;
  pin(groups.d, groups.m, groups.s, tiles.d, tiles.m, tiles.s, q, sq_b, sq_h, sq_t, idx, lengths, parts0, parts1, nparts);
  pin(shape.l, shape.nslots, shape.lprime, shape.window, shape.d.m, shape.d.s, a.blocks.m, a.blocks.s, hpg, Tq, scale, a.part_ml, a.part_o);
  const int bg = blockIdx.y, b = groups.div(bg), grp = bg - b * groups.d;
  const int ti = tiles.div(blockIdx.z), ht = blockIdx.z - ti * tiles.d;
  const int len = scalar_load(lengths, b);

  // The tile's queries to LDS, on their way while the length is: row by row here, as a lane's quarters of
  // rows below, where every 16 bytes straight from memory would be a cache line of their own.
  constexpr int QP = DK * (int)sizeof(S) + 16, QL = DK * (int)sizeof(S) / 16;  // row pitch, 16-byte pieces of a row
  constexpr int NQ = (16 * QL + 64 * NW - 1) / (64 * NW);
  uint4 qx[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int e = min(i * 64 * NW + (int)threadIdx.x, 16 * QL - 1), c = e / QL;
    const S* qp = reinterpret_cast<const S*>(q) + b * sq_b + (int64_t)(grp * hpg + min(ht * 16 + c, hpg - 1)) * sq_h + ti * sq_t;
    qx[i] = *reinterpret_cast<const uint4*>(qp + (e - c * QL) * (16 / (int)sizeof(S)));
  }
  int64_t chosen = -1;
  if (parts1 && lane < shape.nslots) chosen = idx[((int64_t)bg * Tq + ti) * shape.nslots + lane];
  float z[3] = {0.f, 0.f, 0.f};  // the gate inputs of column c16's head
  if (WHOLE && a.gates) {
    const S* zp = reinterpret_cast<const S*>(a.gates) + b * a.sg_b + (int64_t)(grp * hpg + min(ht * 16 + c16, hpg - 1)) * a.sg_h + ti * a.sg_t;
#pragma unroll
    for (int i = 0; i < 3; ++i) z[i] = Elem<T>::to_f32(zp[i * a.sg_k]);
  }
  const int p = max(len, 0) - Tq + ti;

  // The wave's source, and its tiles of the source's key list: from begin on, every step-th key.
  int s, begin, end, step, w_lo, w_hi;  // [w_lo, w_hi): the waves of the same source
  int base;
  if constexpr (WHOLE) {
    const int parts2 = nparts - parts0 - parts1;
    const int n0 = parts0 ? kv4_keys(shape, 0, a.src[0].cap, p, &base) : 0;
    const int n1 = parts1 ? kv4_keys(shape, 1, a.src[1].cap, p, &base) : 0;
    const int n2 = parts2 ? kv4_keys(shape, 2, a.src[2].cap, p, &base) : 0;
    // waves by keys, at least one for a source that has any
    const float each = (float)NW / fmaxf((float)n0 + (float)n1 + (float)n2, 1.f);
    const int most0 = NW - (n1 > 0) - (n2 > 0);
    const int w0 = __builtin_amdgcn_readfirstlane(n0 == 0 ? 0 : n1 + n2 == 0 ? NW : min(max((int)rintf((float)n0 * each), 1), most0));
    const int w1 = __builtin_amdgcn_readfirstlane(n1 == 0 ? 0 : n2 == 0 ? NW - w0 : min(max((int)rintf((float)n1 * each), 1), NW - w0 - 1));
    s = wave < w0 ? 0 : wave < w0 + w1 ? 1 : 2;
    if (n0 + n1 + n2 == 0) s = parts0 ? 0 : parts1 ? 1 : 2;  // (one that is there)
    w_lo = s == 0 ? 0 : s == 1 ? w0 : w0 + w1;
    w_hi = s == 0 ? w0 : s == 1 ? w0 + w1 : NW;
    end = s == 0 ? n0 : s == 1 ? n1 : n2;
    begin = (wave - w_lo) * kKvTile;
    step = (w_hi - w_lo) * kKvTile;
  } else {
    s = (int)blockIdx.x < parts0 ? 0 : (int)blockIdx.x < parts0 + parts1 ? 1 : 2;
    w_lo = 0, w_hi = NW;
    step = NW * kKvTile;
  }
  const Kv4Source src = a.src[s];
  const Kv4Pages pg = src.pg;
  pin(pg.k, pg.ks, pg.v, pg.vs, pg.n_pages, pg.shift, src.tables, src.st_b, src.W, src.cap, src.parts.d, src.parts.m, src.parts.s);
  const int keys = kv4_keys(shape, s, src.cap, p, &base);
  if constexpr (!WHOLE) {
    const int part = blockIdx.x - (s > 0 ? parts0 : 0) - (s > 1 ? parts1 : 0);
    const int each = kv4_part_keys(keys, src.parts);
    const int64_t from = (int64_t)part * each;
    if (from >= keys) return;  // nothing here
    begin = (int)from + wave * kKvTile, end = min(keys - (int)from, each) + (int)from;
  }
  const int first = s == kDecWin ? p + 1 - min(shape.window, p + 1) : 0;  // keys below are masked
  const int last = s == kDecCmp ? keys - 1 : p;                           // keys above are masked

  int lv = chosen < 0 ? -1 : (int)(chosen < INT_MAX ? chosen : INT_MAX);  // lane i: the block of slot i, once
  if (s == kDecSel) {
    if (__ballot(lv >= 0) == 0 && lane == 0) lv = p / shape.lprime;  // no block chosen: the query's own
    bool again = false;
    for (int i = 0; i + 1 < shape.nslots; ++i) again |= lane > i && lv == __builtin_amdgcn_readlane(lv, i);
    if (again) lv = -1;
  }
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int e = i * 64 * NW + threadIdx.x, c = e / QL;
    if (16 * QL % (64 * NW) == 0 || e < 16 * QL) *reinterpret_cast<uint4*>(s_buf + c * QP + (e - c * QL) * 16) = qx[i];
  }
  __syncthreads();
  uint32_t qf[NS][NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint4* qp = reinterpret_cast<const uint4*>(s_buf + c16 * QP + (g4 * (DK / 4) + 8 * j) * (int)sizeof(S));
    if constexpr (NS == 1) {
      const uint4 x = qp[0];
      qf[0][j][0] = x.x, qf[0][j][1] = x.y, qf[0][j][2] = x.z, qf[0][j][3] = x.w;
    } else {
      const uint4 xy[2] = {qp[0], qp[1]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = xy[i >> 1];
        uint32_t w[NS];
        split_pair<NS>(__uint_as_float(i & 1 ? x.z : x.x), __uint_as_float(i & 1 ? x.w : x.y), w);
#pragma unroll
        for (int n = 0; n < NS; ++n) qf[n][j][i] = w[n];
      }
    }
  }
  __syncthreads();  // V's rows go over the queries
  const int* tab = src.tables + b * src.st_b;

  f32x4 oacc[DV / 16];
#pragma unroll
  for (int j = 0; j < DV / 16; ++j) oacc[j] = zero4();
  // reference of the lane's column (log2 units; the running maximum, or up to 8 below it) and the
  // lane's share of the sum
  float ref = -INFINITY, ls = 0.f;
  // a negative scale goes to the queries' signs, so that the largest product is the largest score; a
  // scale of 0 is the smallest number, which leaves a masked key at -inf
  const float scale2 = scale == 0.f ? FLT_MIN : fabsf(scale) * kLog2e;
  if (scale < 0.f) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[n][j][i] ^= 0x80008000u;
  }
  uint16_t* vs = reinterpret_cast<uint16_t*>(s_buf) + wave * kKvTile * VP;

  for (int pos = begin; pos < end; pos += 32 * step) {
    // Where the wave's next 32 tiles lie, two 16-key groups each, one a lane: the group's row of the
    // pool over 16, and the keys [lo, hi) of it that are visible
    const int nt = min((int)((uint32_t)(end - pos + step - 1) / (uint32_t)step), 32);
    int row16 = 0, vis = 0;
    {
      const int e = pos + (lane >> 1) * step + (lane & 1) * 16;
      int64_t k0 = base + e;
      bool ok = (lane >> 1) < nt && e < end;
      if (s == kDecSel) {
        const int slot = ok ? a.blocks.div(e) : 0;
        const int blk = __shfl(lv, slot);
        k0 = (int64_t)blk * shape.lprime + (e - slot * shape.lprime);
        ok = ok && blk >= 0 && k0 <= last;
      }
      const int64_t j = k0 >> pg.shift;
      int page = -1;
      if (ok && j < src.W) page = tab[j];
      if (page >= 0 && page < pg.n_pages) {
        row16 = ((page * groups.d + grp) << (pg.shift - 4)) + (((int)k0 & ((1 << pg.shift) - 1)) >> 4);
        const int lo = max(0, first - (int)k0), hi = min(16, last + 1 - (int)k0);
        vis = lo < hi ? lo | hi << 8 : 0;
      }
    }
    // Addresses as a wave's base and a lane's constant offset: the wide products and sums stay
    // scalar.  (Left to itself the compiler adds base and offset first, and the row to that a lane.)
    Tile t;
    auto load_k = [&](int i) __attribute__((always_inline)) {
      const int64_t r0 = __builtin_amdgcn_readlane(row16, 2 * i), r1 = __builtin_amdgcn_readlane(row16, 2 * i + 1);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const wave_ptr kb = wave_base(pg.k, (u ? r1 : r0) * (16 * DK / 2)), sb = wave_base(pg.ks, (u ? r1 : r0) * (16 * DK / 32));
        const uint32_t ko = c16 * (DK / 2) + g4 * (DK / 8), so = c16 * (DK / 32) + g4 * (DK / 4) / 32;
        if constexpr (NJ % 4 == 0) {
          const u32x4 w = load_at<u32x4>(kb, ko);
#pragma unroll
          for (int j = 0; j < NJ; ++j) t.k[u][j] = w[j & 3];
        } else if constexpr (NJ % 2 == 0) {
#pragma unroll
          for (int j = 0; j < NJ; j += 2) {
            const u32x2 w = load_at<u32x2>(kb, ko + 4 * j);
            t.k[u][j] = w[0], t.k[u][j + 1] = w[1];
          }
        } else {
          t.k[u][0] = load_at<uint32_t>(kb, ko);
        }
        t.ks[u][0] = load_at<uint8_t>(sb, so);
        if constexpr (DK == 192) t.ks[u][1] = load_at<uint8_t>(sb, so + 1);  // the quarter's second block
      }
    };
    auto load_v = [&](int i) __attribute__((always_inline)) {
      const int64_t r0 = __builtin_amdgcn_readlane(row16, 2 * i), r1 = __builtin_amdgcn_readlane(row16, 2 * i + 1);
#pragma unroll
      for (int i2 = 0; i2 < NV; ++i2) {
        const int r = ((i2 * 64 + lane) / LPR) % kKvTile, blk = lane % LPR;
        if constexpr (LPR == 4) {  // a load is one group of keys
          const int64_t rv = i2 ? r1 : r0;
          t.v[i2] = __builtin_bit_cast(uint4, load_at<u32x4>(wave_base(pg.v, rv * (16 * DV / 2)), (r & 15) * (DV / 2) + blk * 16));
          t.vs[i2] = load_at<uint8_t>(wave_base(pg.vs, rv * (16 * DV / 32)), (r & 15) * (DV / 32) + blk);
        } else {
          const int64_t rw = (r & 16 ? r1 : r0) * 16 + (r & 15);
          t.v[i2] = *reinterpret_cast<const uint4*>(pg.v + rw * (DV / 2) + blk * 16);
          t.vs[i2] = pg.vs[rw * (DV / 32) + blk];
        }
      }
    };
    // One tile's registers: V's take the next tile's rows once they are in LDS, K's once the scores
    // are, so that those are on their way through the softmax and the second product; the waves
    // that fit beside each other hide the rest.  (Two tiles' registers: three waves a SIMD at dk = 192
    // instead of four.)  Past the last tile they are the pool's first rows, unused.
    load_v(0);
    load_k(0);
    for (int i = 0; i < nt; ++i) {
      const int v0 = __builtin_amdgcn_readlane(vis, 2 * i), v1 = __builtin_amdgcn_readlane(vis, 2 * i + 1);
      const bool full = v0 == 16 << 8 && v1 == 16 << 8;
      // V rows to LDS as bf16; rows that are not visible are zeros, so that what they hold never
      // meets a zero probability
#pragma unroll
      for (int i2 = 0; i2 < NV; ++i2) {
        const int r = (i2 * 64 + lane) / LPR, blk = lane % LPR;
        if (!full) {
          const int vv = r & 16 ? v1 : v0, rr = r & 15;
          const bool in = rr >= (vv & 255) && rr < vv >> 8;
          const uint32_t keep = in ? ~0u : 0u;
          t.v[i2] = make_uint4(t.v[i2].x & keep, t.v[i2].y & keep, t.v[i2].z & keep, t.v[i2].w & keep);
          t.vs[i2] = in ? t.vs[i2] : 127u;
        }
        if (kKvTile * LPR >= 64 || r < kKvTile) {
          const uint4 w = t.v[i2];
          const float sc = e8m0(t.vs[i2]);
          uint16_t* dst = vs + r * VP + blk * 32;
          *reinterpret_cast<uint4*>(dst) = fp4x8_to_bf16(w.x, sc);
          *reinterpret_cast<uint4*>(dst + 8) = fp4x8_to_bf16(w.y, sc);
          *reinterpret_cast<uint4*>(dst + 16) = fp4x8_to_bf16(w.z, sc);
          *reinterpret_cast<uint4*>(dst + 24) = fp4x8_to_bf16(w.w, sc);
        }
      }
      load_v(min(i + 1, 31));
      f32x4 st[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        st[u] = zero4();
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint4 kf = fp4x8_to_bf16(t.k[u][j], e8m0(kv4_scale<DK>(t.ks[u][0], t.ks[u][DK == 192], j, g4)));
#pragma unroll
          for (int n = 0; n < NS; ++n)
            st[u] = Mma<bf16>::run(st[u], kf, make_uint4(qf[n][j][0], qf[n][j][1], qf[n][j][2], qf[n][j][3]));
        }
      }
      load_k(min(i + 1, 31));
      // softmax: lane holds head c16, keys 4 g4 + i of each group
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!full) {
          const int vv = u ? v1 : v0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = 4 * g4 + k;
            st[u][k] = r >= (vv & 255) && r < vv >> 8 ? st[u][k] : -INFINITY;
          }
        }
      }
      float m = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                      fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
      m = wave_max16(m) * scale2;
      if (__ballot(m > ref + kLazyRescale)) {  // a maximum well above the reference: it moves
        const float now = fmaxf(ref, m);
        const float corr = ref == -INFINITY ? 0.f : fast_exp2(ref - now);
        ref = now;
        ls *= corr;
#pragma unroll
        for (int j = 0; j < DV / 16; ++j) oacc[j] *= corr;
      }
      const float nref = ref == -INFINITY ? 0.f : ref;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          st[u][k] = fast_exp2(fmaf(st[u][k], scale2, -nref));
          ls += st[u][k];
        }
      uint32_t pw[4][NS];
      split_pair<NS>(st[0][0], st[0][1], pw[0]);
      split_pair<NS>(st[0][2], st[0][3], pw[1]);
      split_pair<NS>(st[1][0], st[1][1], pw[2]);
      split_pair<NS>(st[1][2], st[1][3], pw[3]);
      wave_lds_sync();
      const uint16_t* vt = vs + (4 * g4 + (c16 >> 2)) * VP + (c16 & 3) * 4;
#pragma unroll
      for (int j = 0; j < DV / 16; ++j) {
        const uint4 vf = ld_tr_pair(vt + 16 * j, 16 * VP);
#pragma unroll
        for (int n = 0; n < NS; ++n)
          oacc[j] = Mma<bf16>::run(oacc[j], vf, make_uint4(pw[0][n], pw[1][n], pw[2][n], pw[3][n]));
      }
      wave_lds_sync();  // the tile's reads are done before the next one's rows are written
    }
  }
  ls = wave_sum16(ls);

  // The waves' states merged through LDS, over the V rows once every wave is past them: each brings its O
  // to its source's maximum (WHOLE: on to the source's share of out), then they are added up.
  if (g4 == 0) {
    s_m[wave][c16] = ref;
    s_l[wave][c16] = ls;
  }
  __syncthreads();
  float M = -INFINITY, l = 0.f;  // column c16's maximum and sum
  for (int w = w_lo; w < w_hi; ++w) M = fmaxf(M, s_m[w][c16]);
  for (int w = w_lo; w < w_hi; ++w) {
    const float m = s_m[w][c16];
    l += (m == -INFINITY ? 0.f : fast_exp2(m - M)) * s_l[w][c16];
  }
  float own = ref == -INFINITY ? 0.f : fast_exp2(ref - M);
  const int64_t at = ((int64_t)bg * gridDim.z + blockIdx.z) * nparts + blockIdx.x;
  const int nc = min(16, hpg - ht * 16);  // the tile's heads
  if constexpr (WHOLE) {
    // no visible key: 0 (the sum is exactly 0); a NaN sum is one of a visible key and stays
    own *= l == 0.f ? 0.f : (a.gates ? kv4_gate(a.act, s, z[0], z[1], z[2]) : 1.f) / l;
  } else if (threadIdx.x < nc) {
    *reinterpret_cast<float2*>(a.part_ml + (at * 16 + c16) * 2) = make_float2(M, l);
  }
  float* so = reinterpret_cast<float*>(s_buf);
#pragma unroll
  for (int j = 0; j < DV / 16; ++j)
    *reinterpret_cast<f32x4*>(so + (wave * 16 + c16) * OP + 16 * j + 4 * g4) = oacc[j] * own;
  __syncthreads();
  for (int e = threadIdx.x; e < nc * (DV / 4); e += 64 * NW) {
    const int c = e / (DV / 4), f = 4 * (e % (DV / 4));
    f32x4 o = *reinterpret_cast<const f32x4*>(so + c * OP + f);
#pragma unroll
    for (int w = 1; w < NW; ++w) o += *reinterpret_cast<const f32x4*>(so + (w * 16 + c) * OP + f);
    if constexpr (WHOLE)
      store4<T>(reinterpret_cast<S*>(a.out) + b * a.so_b + (int64_t)(grp * hpg + ht * 16 + c) * a.so_h + ti * a.so_t + f, o);
    else
      *reinterpret_cast<f32x4*>(a.part_o + at * 16 * DV + c * DV + f) = o;
  }
}

// The join of a row's parts: out = sum_i w_i O_i, the weight of part i of source s being gate_s
// exp2(m_i - M_s) / L_s with M_s the source's largest maximum and L_s = sum_i exp2(m_i - M_s) l_i.
//
// WAVES a (head, query row, request): each wave works out every weight, a part a lane, and adds up
// every WAVES-th part, DV / 64 features a lane.  Bound by the latency of length -> {m, l} -> O.  One wave
// up to kMixFew parts, sixteen beyond.  Call of 16 heads, bf16 dk 192, one wave / sixteen in us: 16 parts
// of 16 rows 9.8 / 10.8, of 512 rows 15.0 / 17.8; 21 of 384 14.1 / 17.2; 32 of 16 11.2 / 10.8, of 256 15.0 / 14.6;
// 64 of 16 14.7 / 11.0.
constexpr int kMixFew = 24, kMixMost = 512;  // (three more by rounding)

template <typename T, int DV, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void kv4_mix_kernel(Kv4Attn a) {
  using S = typename Store<T>::type;
  constexpr int FPL = DV >= 64 ? DV / 64 : 1;                // features of a lane
  constexpr int NL = WAVES == 1 ? 1 : (kMixMost + 3 + 63) / 64;  // parts of a lane, at most
  typedef float vf __attribute__((ext_vector_type(FPL)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const IntDiv heads = a.heads, rows = a.rows, hpgd = a.hpgd;
  const Kv4Shape shape{a.l, a.nslots, a.lprime, a.window, a.d};
  const int nparts = a.nparts, Tq = a.Tq, G = a.G, nht = a.tiles.d, parts0 = a.parts[0], parts1 = a.parts[1];
  const int* lengths = a.lengths;
  pin(heads.d, heads.m, heads.s, rows.d, rows.m, rows.s, hpgd.d, hpgd.m, hpgd.s, shape.l, shape.nslots, shape.lprime,
      shape.window, shape.d.m, shape.d.s, nparts, Tq, G, nht, parts0, parts1, lengths);
  pin(a.gates, a.sg_b, a.sg_h, a.sg_t, a.sg_k, a.act, a.part_ml, a.part_o, a.src[0].cap, a.src[1].cap, a.src[2].cap, a.out,
      a.so_b, a.so_h, a.so_t, a.n_rows);
  // row = (b Tq + ti) H + h
  const int row = WAVES == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x;
  if (row >= a.n_rows) return;
  const int bt = heads.div(row), h = row - bt * heads.d, b = rows.div(bt), ti = bt - b * rows.d;
  const int grp = hpgd.div(h), hc = h - grp * hpgd.d, c = hc & 15;
  const int p = max(scalar_load(lengths, b), 0) - Tq + ti;
  const int64_t at = ((int64_t)(b * G + grp) * (Tq * nht) + ti * nht + (hc >> 4)) * nparts;

  float gate[3] = {1.f, 1.f, 1.f};
  if (a.gates) {
    const S* z = reinterpret_cast<const S*>(a.gates) + b * a.sg_b + h * a.sg_h + ti * a.sg_t;
    const float z0 = Elem<T>::to_f32(z[0]), z1 = Elem<T>::to_f32(z[a.sg_k]), z2 = Elem<T>::to_f32(z[2 * a.sg_k]);
#pragma unroll
    for (int s = 0; s < 3; ++s) gate[s] = kv4_gate(a.act, s, z0, z1, z2);
  }
  int n[3];  // the sources' parts that hold keys
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    int base;
    const int keys = kv4_keys(shape, s, a.src[s].cap, p, &base);
    const int each = kv4_part_keys(keys, a.src[s].parts);
    n[s] = keys && (s == 0 ? parts0 : s == 1 ? parts1 : nparts - parts0 - parts1) ? (int)((uint32_t)(keys + each - 1) / (uint32_t)each) : 0;
  }
  // lane: {m, l} of parts lane, lane + 64, ... of the row's
  float m[NL], l[NL], w[NL];
  int src[NL];
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at * 16 + c;
#pragma unroll
  for (int k = 0; k < NL; ++k) {
    const int i = 64 * k + lane;
    const int s = i < parts0 ? 0 : i < parts0 + parts1 ? 1 : 2;
    const int k0 = i - (s > 0 ? parts0 : 0) - (s > 1 ? parts1 : 0);
    const bool on = i < nparts && k0 < (s == 0 ? n[0] : s == 1 ? n[1] : n[2]);
    src[k] = on ? s : 3;
    const float2 x = on ? ml[(int64_t)i * 16] : make_float2(-INFINITY, 0.f);
    m[k] = x.x, l[k] = x.y, w[k] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    if (n[s] == 0) continue;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int k = 0; k < NL; ++k) M = fmaxf(M, src[k] == s ? m[k] : -INFINITY);
    M = wave_butterfly(M, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const float e = m[k] == -INFINITY ? 0.f : fast_exp2(m[k] - M);
      if (src[k] == s) L += e * l[k], w[k] = e;
    }
    L = wave_butterfly(L, [](float x, float y) { return x + y; });
    // no visible key: 0 (the sum is exactly 0); a NaN sum is one of a visible key and stays
    const float g = L == 0.f ? 0.f : gate[s] / L;
#pragma unroll
    for (int k = 0; k < NL; ++k)
      if (src[k] == s) w[k] *= g;
  }
  vf o{};
  const float* po = a.part_o + at * 16 * DV + c * DV + FPL * (lane & (DV / FPL - 1));
#pragma unroll
  for (int k = 0; k < NL; ++k) {
    uint64_t left = __ballot(src[k] != 3);
    if constexpr (WAVES > 1) left &= 0x0001000100010001ull << wave;  // i = wave mod 16
    while (left) {  // four parts at once
      int i[4];
      float x[4];
      vf y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool some = left != 0;
        i[u] = some ? __builtin_ctzll(left) : i[0];
        x[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w[k]), i[u]));
        if (!some) x[u] = 0.f;
        left &= left - 1;
        y[u] = *reinterpret_cast<const vf*>(po + (int64_t)(64 * k + i[u]) * 16 * DV);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) o += x[u] * y[u];
    }
  }
  if constexpr (WAVES > 1) {
    __shared__ vf s_o[WAVES][64];
    s_o[wave][lane] = o;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 1; i < WAVES; ++i) o += s_o[i][lane];
  }
  if (lane < DV / FPL) {
    S* dst = reinterpret_cast<S*>(a.out) + b * a.so_b + (int64_t)h * a.so_h + ti * a.so_t + FPL * lane;
#pragma unroll
    for (int k = 0; k < FPL; ++k) dst[k] = Elem<T>::from_f32(o[k]);
  }
}

template <typename T, int DK, int DV>
static void launch_kv4(const Kv4Attn& a, hipStream_t st) {
  const int nht = (a.hpg + 15) / 16;
  if (a.whole) {
    constexpr int NW = kv4_whole_waves(sizeof(typename Store<T>::type), DK);
    hipLaunchKernelGGL((kv4_attn_kernel<T, DK, DV, NW, true>), dim3(1, a.B * a.G, a.Tq * nht), dim3(64 * NW), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((kv4_attn_kernel<T, DK, DV, kKvWaves, false>), dim3(a.nparts, a.B * a.G, a.Tq * nht), dim3(64 * kKvWaves), 0, st, a);
  if (a.nparts <= kMixFew)
    hipLaunchKernelGGL((kv4_mix_kernel<T, DV, 1>), dim3((a.n_rows + 3) / 4), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv4_mix_kernel<T, DV, 16>), dim3(a.n_rows), dim3(1024), 0, st, a);
}

// Parts of each source: a round of keys or more a part, and two workgroups a CU in all.  Call in us with
// 256 / 384 / 512 / 768 / 1024: 131072 keys of H64 G4 dk 192 28.8 / 27.9 / 26.3 / 29.4 / 31.9; 16 requests through three
// sources at H32 G2 dk 128 13.9 / 14.9 / 14.5 / 15.7 / 29.2; four fp32 requests of four rows, H16 G4 dk 64, up
// to 5000 keys 13.7 / 12.6 / 12.7 / 11.4 / 14.6.
constexpr int64_t kKvGroups = 512;
static_assert(kKvGroups <= kMixMost);
static void kv4_split(const nsa_kv4_attn_args& x, Kv4Attn& a) {
  const int64_t columns = (int64_t)a.B * a.G * a.Tq * ((a.hpg + 15) / 16);
  int64_t keys[3] = {0, 0, 0}, all = 0;
  for (int s = 0; s < 3; ++s) {
    if (!a.parts[s]) continue;
    const int64_t cap = std::min(a.src[s].cap, x.max_length);
    keys[s] = s == kDecSel   ? (int64_t)a.nslots * a.lprime
              : s == kDecCmp ? std::min(a.src[s].cap, x.max_length >= a.l ? (x.max_length - a.l) / x.d + 1 : 0)
                             : std::min<int64_t>((int64_t)a.window + 15, cap);
    all += keys[s] = std::max<int64_t>(keys[s], 1);
  }
  const int64_t most = std::max<int64_t>(1, kKvGroups / columns);
  a.nparts = 0;
  for (int s = 0; s < 3; ++s) {
    if (!a.parts[s]) continue;
    const int64_t share = std::max<int64_t>(1, keys[s] * most / all);
    a.parts[s] = (int)std::min<int64_t>((keys[s] + kKvStep - 1) / kKvStep, share);
    a.src[s].parts = IntDiv::make(a.parts[s]);
    a.nparts += a.parts[s];
  }
  // A workgroup for a row's whole work, or parts and their join?  Whole is one launch, 4 us less of the host,
  // and no partials, but a row's keys then go 512 a round (fp32 from dk 128 on 256) however many CUs are
  // idle.  Call, whole / parts in us, bf16 dk 192: 64 columns of 1024 keys 11.7 / 12.6, of 2048 15.9 / 14.2;
  // 128 columns of 2048 16.6 / 17.6, of 4096 24.2 / 22.8; 256 columns of 4096 31.7 / 33.9.  So whole up to some
  // 22 keys for each column, and with a column a CU or more at any length, where lengths are within a 16th of
  // the longest (256 columns of up to 16384 77 / 86, 512 141 / 163; fp32 dk 128 103 / 105, 203 / 205).  Of few
  // columns up to 1024 keys (bf16 to dk 64 2048) for the host's sake (1024 keys, 4 columns: calls in a row
  // 10.7 / 14.9, one alone 27.6 / 27.8, replayed 11.4 / 9.1).
  // The rule sees the columns and the longest length alone, so that one long request among many short ones
  // gets few workgroups: 131072 keys (H64 G4 bf16 dk 192) alone 26 us, among 16 requests 129, 32 248, 64 482.
  const int64_t few = x.dtype == NSA_BF16 && x.head_dim_qk <= 64 ? 2048 : 1024;
  a.whole = columns >= 256 || all <= std::max<int64_t>(few, 22 * columns);
}

// The call's shape checked; the part of Kv4Attn that the split needs.
static int kv4_attn_shape(const nsa_kv4_attn_args& x, Kv4Attn& a) {
  if (x.dtype != NSA_F32 && x.dtype != NSA_BF16) return set_error(NSA_ERR_INVALID, "dtype not supported");
  if (x.Z < 1 || x.H < 1 || x.n_kv_groups < 1 || x.H % x.n_kv_groups || x.n_ctx_q < 1 || x.max_length < 1)
    return set_error(NSA_ERR_INVALID, "bad shape");
  if (!nsa_head_dims_supported(x.dtype, x.head_dim_qk, x.head_dim_v))
    return set_error(NSA_ERR_UNSUPPORTED, "no kernel for these head dims");
  a.B = x.Z;
  a.G = x.n_kv_groups;
  a.hpg = x.H / x.n_kv_groups;
  a.Tq = x.n_ctx_q;
  if ((int64_t)x.Z * x.n_kv_groups > 65535 || (int64_t)x.n_ctx_q * ((a.hpg + 15) / 16) > 65535 || x.Z > 65535)
    return set_error(NSA_ERR_INVALID, "more than 65535 (request, group) pairs or query row tiles");
  if ((int64_t)x.Z * x.n_ctx_q * x.H > INT_MAX) return set_error(NSA_ERR_INVALID, "more than 2^31 - 1 query rows");
  a.l = x.l;
  a.nslots = x.n_slots;
  a.lprime = x.block_size_selection;
  a.window = x.window_size;
  a.act = x.gate_act;
  a.scale = x.sm_scale;
  int present = 0;
  for (int s = 0; s < 3; ++s) {
    a.parts[s] = 0;
    if (!x.pages[s]) continue;
    ++present;
    if (int rc = kv4_check_pages(x.pages[s], x.n_kv_groups, &a.src[s].pg)) return rc;
    if (x.table_width[s] < 1 || (int64_t)x.table_width[s] << a.src[s].pg.shift > kPagedMaxTokens)
      return set_error(NSA_ERR_INVALID, "a block table of no entries or more than 2^30 tokens");
    if ((int64_t)x.pages[s]->n_pages * x.n_kv_groups * (x.pages[s]->page_size / 16) > INT_MAX)
      return set_error(NSA_ERR_INVALID, "a pool of 2^35 rows or more");
    a.src[s].W = x.table_width[s];
    a.src[s].cap = a.src[s].W << a.src[s].pg.shift;
    a.parts[s] = 1;
  }
  if (!present) return set_error(NSA_ERR_INVALID, "no source");
  if (x.pages[1] && x.pages[2] && x.tables[1] && x.tables[1] == x.tables[2] && a.src[1].pg.shift != a.src[2].pg.shift)
    return set_error(NSA_ERR_INVALID, "one block table for pools of different page sizes");
  if (x.pages[0] && (x.l < 1 || x.d < 1)) return set_error(NSA_ERR_INVALID, "bad l or d");
  if (x.pages[1] && (x.n_slots < 1 || x.n_slots > 64 || x.block_size_selection < 16 ||
                       x.block_size_selection % 16 || x.block_size_selection > (1 << 20)))
    return set_error(NSA_ERR_INVALID, "n_slots outside [1, 64] or block_size_selection no multiple of 16");
  if (x.pages[2] && x.window_size < 1) return set_error(NSA_ERR_INVALID, "window_size < 1");
  if (x.gates ? x.gate_act < 0 || x.gate_act > 2 : present != 1)
    return set_error(NSA_ERR_INVALID, "gate_act outside [0, 2], or several sources without gates");
  a.groups = IntDiv::make(a.G);
  a.heads = IntDiv::make(x.H);
  a.rows = IntDiv::make(a.Tq);
  a.hpgd = IntDiv::make(a.hpg);
  a.n_rows = a.B * a.Tq * x.H;
  a.tiles = IntDiv::make((a.hpg + 15) / 16);
  a.blocks = IntDiv::make(x.pages[1] ? x.block_size_selection : 1);
  a.d = IntDiv::make(x.pages[0] ? x.d : 1);
  kv4_split(x, a);
  return NSA_OK;
}

// parts of all query row tiles
static size_t kv4_attn_parts(const Kv4Attn& a) {
  return a.whole ? 0 : (size_t)a.B * a.G * a.Tq * ((a.hpg + 15) / 16) * a.nparts;
}
static size_t kv4_attn_bytes(const Kv4Attn& a, int dv) { return kv4_attn_parts(a) * 16 * (dv + 2) * 4; }

}  // namespace nsa

using namespace nsa;

extern "C" size_t nsa_kv4_attn_workspace_size(const nsa_kv4_attn_args* x) {
  Kv4Attn a{};
  if (!x || kv4_attn_shape(*x, a)) return 0;
  return kv4_attn_bytes(a, x->head_dim_v);
}

extern "C" int nsa_kv4_attn(const nsa_kv4_attn_args* x, void* ws, size_t ws_bytes, nsa_stream_t stream) {
  if (!x) return set_error(NSA_ERR_INVALID, "args is null");
  Kv4Attn a{};
  if (int rc = kv4_attn_shape(*x, a)) return rc;
  if (!x->q || !x->out || !x->lengths || (x->pages[1] && !x->indices)) return set_error(NSA_ERR_INVALID, "null tensor");
  for (int s = 0; s < 3; ++s)
    if (a.parts[s] && !x->tables[s]) return set_error(NSA_ERR_INVALID, "null block table");
  const int es = x->dtype == NSA_F32 ? 4 : 2;
  auto rows = [&](const void* p, int64_t sz, int64_t sh, int64_t st) {
    return ((uintptr_t)p) % 16 == 0 && (x->Z == 1 || (sz * es) % 16 == 0) && (x->H == 1 || (sh * es) % 16 == 0) &&
           (x->n_ctx_q == 1 || (st * es) % 16 == 0);
  };
  if (!rows(x->q, x->stride_qz, x->stride_qh, x->stride_qt) || !rows(x->out, x->stride_oz, x->stride_oh, x->stride_ot))
    return set_error(NSA_ERR_LAYOUT, "q and out need 16-byte aligned rows");
  const size_t need = kv4_attn_bytes(a, x->head_dim_v);
  if (ws_bytes < need || (need && (!ws || ((uintptr_t)ws) % 16))) {
    char msg[128];
    snprintf(msg, sizeof(msg), "workspace of %zu bytes (16-byte aligned) required, %zu given", need, ws_bytes);
    return set_error(NSA_ERR_WORKSPACE, msg);
  }
  a.q = x->q;
  a.sq_b = x->stride_qz, a.sq_h = x->stride_qh, a.sq_t = x->stride_qt;
  a.out = x->out;
  a.so_b = x->stride_oz, a.so_h = x->stride_oh, a.so_t = x->stride_ot;
  a.gates = x->gates;
  a.sg_b = x->stride_gz, a.sg_h = x->stride_gh, a.sg_t = x->stride_gt, a.sg_k = x->stride_gk;
  a.idx = x->indices;
  a.lengths = x->lengths;
  for (int s = 0; s < 3; ++s) {
    a.src[s].tables = x->tables[s];
    a.src[s].st_b = x->stride_table[s];
  }
  a.part_ml = static_cast<float*>(ws);
  a.part_o = a.part_ml + kv4_attn_parts(a) * 32;
#define NSA_CASE(DKV, DVV)                                                               \
  if (x->head_dim_qk == DKV && x->head_dim_v == DVV) {                                   \
    if (x->dtype == NSA_F32) launch_kv4<float, DKV, DVV>(a, (hipStream_t)stream);        \
    else launch_kv4<bf16, DKV, DVV>(a, (hipStream_t)stream);                             \
    return hipGetLastError() == hipSuccess ? NSA_OK : set_error(NSA_ERR_HIP, "kv4 attention launch failed"); \
  }
  NSA_HEAD_DIMS(NSA_CASE)
#undef NSA_CASE
  return set_error(NSA_ERR_UNSUPPORTED, "no kernel for these head dims");
}
