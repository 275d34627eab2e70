// gmoe_attn8.hip — the paged KV cache held in 8 bits: append, attention, reading back.
//
// A sequence's positions are cut into blocks of 16. Of a complete block, one kv head's keys
// (values) x are held as codes c = rint(x * 127 / m), m = max |x| over the block's 16 rows,
// and a scale s = m / 127 rounded to f32; they stand for c * s. The block of the sequence's
// last position is also held in f32 as it was given (keys rotated): a token attends to its
// own block's rows in f32 and to every earlier block's as held in 8 bits, so that its
// context does not depend on how the sequence was cut into calls.
//
// Codes and scales are formed in 64 bits from the f32 rows: at 32, x * 127 / m next to the
// middle between two codes can round to either, and the code would depend on the order of the
// operations. The rotation's angle is formed in 64 bits too (in f32, position 32768 times a
// frequency near 1 is 1e-3 off) and the rotated pair rounded once.
//
// Non-finite input. A block with a NaN or an infinity has the scale NaN, and stands for NaN
// throughout. A NaN or +inf score, or none above -inf, makes a row's weights uniform over its
// span, as with a cache in f32.
#include "gmoe_device.h"

namespace gmoe {

namespace {

// Unit of one block and kv head in a page: keys' codes, then the values'.
__device__ __forceinline__ size_t kv8_block(const Kv8Pool& p, uint32_t page, uint32_t block, uint32_t h) {
  const uint32_t m = p.bs / kKv8Block;
  return ((size_t)page * p.n_kv + h) * m + block % m;
}
__device__ __forceinline__ uint8_t* kv8_codes(const Kv8Pool& p, size_t unit) {
  return p.codes + unit * (2 * kKv8Block) * p.hdp;
}
// Byte of key row r, dim d in its block.
__device__ __forceinline__ uint32_t kv8_key(uint32_t hdp, uint32_t r, uint32_t d) {
  return d < hdp / 64 * 64 ? d / 64 * 1024 + r * 64 + d % 64 : d / 64 * 1024 + r * 32 + d % 64;
}
__device__ __forceinline__ uint32_t kv8_page(const Kv8Pool& p, uint32_t table, uint32_t block) {
  return p.tables[(size_t)table * p.ppseq + block / (p.bs / kKv8Block)];
}
// Open rows of a sequence's kv head: keys, and the values n_kv * 16 * hd floats further on.
__device__ __forceinline__ float* kv8_open(const Kv8Pool& p, uint32_t table, uint32_t h) {
  return p.open + ((size_t)table * 2 * p.n_kv + h) * kKv8Block * p.hd;
}

__device__ __forceinline__ void turn(double turns, uint32_t pos, double& c, double& s) {
  double t = (double)pos * turns;
  t -= rint(t);
  sincospi(2.0 * t, &s, &c);
}
__device__ __forceinline__ float2 rotated(float x, float y, double c, double s) {
  const double a = x, b = y;
  return make_float2((float)(a * c - b * s), (float)(a * s + b * c));
}

// Elements 2j and 2j + 1 of p: sums of nsl slices in slice order.
__device__ __forceinline__ float2 pair_of(const float* p, uint32_t j, uint32_t nsl, uint64_t stride) {
  float2 v = make_float2(p[2 * j], p[2 * j + 1]);
  for (uint32_t g = 1; g < nsl; g++) {
    v.x += p[g * stride + 2 * j];
    v.y += p[g * stride + 2 * j + 1];
  }
  return v;
}

// The 16 rows kt, vt (in LDS, hs floats apart) of one block and head to codes and scales, by 256
// threads; red: 8 words of LDS. Every thread calls it after a barrier that follows the rows'.
__device__ void hold_block(const Kv8Pool& p, size_t unit, const float* kt, const float* vt, uint32_t hs, uint32_t* red) {
  const uint32_t t = threadIdx.x, n = kKv8Block * p.hd;
  uint32_t mk = 0, mv = 0;  // as bits: NaN above infinity above every number
  for (uint32_t x = t; x < n; x += 256) {
    const uint32_t at = x / p.hd * hs + x % p.hd;
    mk = max(mk, __float_as_uint(kt[at]) & 0x7fffffffu);
    mv = max(mv, __float_as_uint(vt[at]) & 0x7fffffffu);
  }
  for (int o = 32; o; o >>= 1) {
    mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
    mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
  }
  if ((t & 63) == 0) {
    red[t >> 6] = mk;
    red[4 + (t >> 6)] = mv;
  }
  __syncthreads();
  mk = max(max(red[0], red[1]), max(red[2], red[3]));
  mv = max(max(red[4], red[5]), max(red[6], red[7]));
  // 127 times 1 / m, as a program without a kernel forms it: on a tie (x = m / 2) the product's last
  // bit decides, and the same operations give the same code
  auto inv = [](uint32_t m) { return m == 0 || m >= 0x7f800000u ? 0.0 : 127.0 * (1.0 / (double)__uint_as_float(m)); };
  auto scale = [](uint32_t m) {
    return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (float)((double)__uint_as_float(m) / 127.0);
  };
  // a NaN's code is any: its block's scale says so
  auto code = [](float x, double i) { return i == 0.0 ? 128u : (uint32_t)((int)rint((double)x * i) + 128) & 255u; };
  const double ik = inv(mk), iv = inv(mv);
  uint8_t* dst = kv8_codes(p, unit);
  for (uint32_t x = t; x < kKv8Block * p.hdp / 4; x += 256) {
    const uint32_t r = x / (p.hdp / 4), d = x % (p.hdp / 4) * 4;
    uint32_t w = 0;
    for (uint32_t b = 0; b < 4; b++) w |= (d + b < p.hd ? code(kt[r * hs + d + b], ik) : 128u) << 8 * b;
    *reinterpret_cast<uint32_t*>(dst + kv8_key(p.hdp, r, d)) = w;
  }
  uint32_t* vd = reinterpret_cast<uint32_t*>(dst + kKv8Block * p.hdp);
  for (uint32_t x = t; x < kKv8Block * p.hdp / 4; x += 256) {
    const uint32_t d = x / 4, r = x % 4 * 4;
    uint32_t w = 0;
    for (uint32_t b = 0; b < 4; b++) w |= (d < p.hd ? code(vt[(r + b) * hs + d], iv) : 128u) << 8 * b;
    vd[x] = w;
  }
  if (t == 0) {
    p.scales[2 * unit] = scale(mk);
    p.scales[2 * unit + 1] = scale(mv);
  }
}

// Rows of one block and kv head, hs floats apart: those below r0 from the open rows, the next n
// from k (rotated) and v, row r being entry ent(r); zeros after them.
template <class F>
__device__ __forceinline__ void block_rows(const Kv8Args& a, uint32_t table, uint32_t block, uint32_t r0, uint32_t n,
                                           uint32_t h, float* kt, float* vt, uint32_t hs, F&& ent) {
  const Kv8Pool& p = a.p;
  const uint32_t t = threadIdx.x, hd = p.hd, half = hd / 2;
  const float* old = kv8_open(p, table, h);
  for (uint32_t x = t; x < r0 * hd; x += 256) {
    const uint32_t at = x / hd * hs + x % hd;
    kt[at] = old[x];
    vt[at] = old[(size_t)p.n_kv * kKv8Block * hd + x];
  }
  for (uint32_t x = t; x < n * half; x += 256) {
    const uint32_t r = r0 + x / half, c = x % half;
    const size_t from = (size_t)ent(r) * a.kv_stride + h * hd;
    double cs, sn;
    turn(p.turns[c], block * kKv8Block + r, cs, sn);
    const float2 k = pair_of(a.k + from, c, a.nsl, a.sl_stride), v = pair_of(a.v + from, c, a.nsl, a.sl_stride);
    reinterpret_cast<float2*>(kt + r * hs)[c] = rotated(k.x, k.y, cs, sn);
    reinterpret_cast<float2*>(vt + r * hs)[c] = v;
  }
  for (uint32_t x = t + (r0 + n) * hd; x < kKv8Block * hd; x += 256) kt[x / hd * hs + x % hd] = vt[x / hd * hs + x % hd] = 0.0f;
}
// The first n rows to the open rows.
__device__ void put_open(const Kv8Pool& p, uint32_t table, uint32_t n, uint32_t h, const float* kt, const float* vt,
                         uint32_t hs) {
  float* to = kv8_open(p, table, h);
  for (uint32_t x = threadIdx.x; x < n * p.hd; x += 256) {
    const uint32_t at = x / p.hd * hs + x % p.hd;
    to[x] = kt[at];
    to[(size_t)p.n_kv * kKv8Block * p.hd + x] = vt[at];
  }
}

// grid (njob, n_kv), 256 threads: a block of the call's positions, one kv head. The job of a
// sequence's first block writes the open rows of its last one, after it has read those that
// were there.
__global__ void __launch_bounds__(256) k8_append(Kv8Args a) {
  extern __shared__ float lds_f[];
  __shared__ uint32_t red[8];
  __shared__ Kv8Job job;
  const Kv8Pool& p = a.p;
  const uint32_t h = blockIdx.y, t = threadIdx.x, n = kKv8Block * p.hd;
  float *kt = lds_f, *vt = kt + n;
  auto rows = [&](uint32_t i) {  // job i, from pinned memory, and its rows
    if (t < sizeof(Kv8Job) / 4) reinterpret_cast<uint32_t*>(&job)[t] = reinterpret_cast<const uint32_t*>(a.hjob + i)[t];
    __syncthreads();
    block_rows(a, job.table, job.block, job.r0, job.n, h, kt, vt, p.hd, [&](uint32_t r) { return job.ent[r]; });
    __syncthreads();
  };
  rows(blockIdx.x);
  const uint32_t flags = job.flags, last = job.last;
  if (h == 0 && a.run)
    for (uint32_t x = blockIdx.x * 256 + t; x < a.nrun; x += gridDim.x * 256) a.run[x] = a.hrun[x];
  if (h == 0 && t == 0 && (flags & kKv8Fresh))
    p.tables[(size_t)job.table * p.ppseq + job.block / (p.bs / kKv8Block)] = job.page;
  if (a.own) {
    float* own = a.own + ((size_t)blockIdx.x * 2 * p.n_kv + h) * n;
    for (uint32_t x = t; x < n; x += 256) {
      own[x] = kt[x];
      own[(size_t)p.n_kv * n + x] = vt[x];
    }
  }
  if (flags & kKv8Whole) hold_block(p, kv8_block(p, job.page, job.block, h), kt, vt, p.hd, red);
  if (!(flags & kKv8First)) return;
  if (last != blockIdx.x) {
    __syncthreads();
    rows(last);
  }
  put_open(p, job.table, job.r0 + job.n, h, kt, vt, p.hd);
}

// ---------------------------------------------------------------------------------
// Attention of few rows: a token of each sequence, or a few tokens of one.
//
// A group is at most 16 (token, query head) rows of one kv head, its tokens in one block of
// one sequence. A workgroup takes one group and one part of its span: part 0 its own block's
// f32 rows (in a step it also appends the token there), part z from 1 on the z-th kKv8Split
// positions of the blocks before it, four waves taking 64 positions at a time in turn.
//
// The products run on v_mfma_f32_16x16x32_f16. A code is an integer of 8 bits, exact in
// fp16: the byte c + 128 under the exponent byte 0x64 is 1024 + c + 128, less 1152 (one
// v_perm and one packed add for two codes). A query row, scaled by a power of two, and a row's
// weights are each the sum of two fp16 (22 bits), two passes each.
//   S^T = K Q^T: row i of the t-th MFMA's A is position 4 t + i % 4 of block i / 4 of the
//     tile's four, so that lane l's 16 scores (column l % 16: the row) are the 16 positions
//     of block l / 16: a block's scale is a lane's scalar;
//   O^T = V^T P^T: those 16 weights are the lane's own B operand as they stand, and the
//     values' 16 bytes a dim are its A operand.
// Codes go from memory to registers as the MFMAs want them, no LDS on the way. The parts' sums
// are joined in a fixed order (k8_join), so a row's bits depend neither on the batch nor on
// how many parts the call has.
// ---------------------------------------------------------------------------------
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t sel) {
  const f16x2 b = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) + b);
}
__device__ __forceinline__ f16x8 codes8(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(f16x8, u32x4{code_pair(lo, 0x04010400u), code_pair(lo, 0x04030402u),
                                         code_pair(hi, 0x04010400u), code_pair(hi, 0x04030402u)});
}
// Eight values as two fp16 each: the first truncated, the second what it leaves, to nearest
// (2^-22 of the value). By the conversion's own builtin: a plain cast of a product is folded
// into one instruction that rounds the product once, and what is left of the product's f32
// value then belongs to another first half.
__device__ __forceinline__ void split8(const float* x, f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]));
#pragma unroll
    for (int j = 0; j < 2; j++) {
      hi[i + j] = h[j];
      lo[i + j] = (_Float16)(x[i + j] - (float)h[j]);
    }
  }
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float max16_32(float v) {  // over the lanes of equal l % 16
  LanePair p = xor16_pair(v);
  p = xor32_pair(fmaxf(p.a, p.b));
  return fmaxf(p.a, p.b);
}
__device__ __forceinline__ float sum16_32(float v) {
  LanePair p = xor16_pair(v);
  p = xor32_pair(p.a + p.b);
  return p.a + p.b;
}
// Exponent of a finite |x| as a power of two at most |x|, at least -100; -100 of anything else.
__device__ __forceinline__ int pow2_of(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 255u) - 127;
  return e == 128 ? -100 : max(e, -100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127

constexpr float kLog2e = 0x1.715476p+0f;
constexpr uint32_t kBadRow = 0x7fc00000u;  // a part's maximum: a NaN or +inf score

// A row's mean over its span, column d: uniform weights (rare). vo: its own block's values.
__device__ float uniform_mean(const Kv8Pool& p, uint32_t table, uint32_t h, uint32_t start, uint32_t pos, uint32_t d,
                              const float* vo, uint32_t vstride) {
  const uint32_t own = pos / kKv8Block * kKv8Block;
  double sum = 0.0;
  for (uint32_t b = start / kKv8Block; b * kKv8Block < own; b++) {
    const size_t u = kv8_block(p, kv8_page(p, table, b), b, h);
    const uint8_t* c = kv8_codes(p, u) + kKv8Block * p.hdp + d * kKv8Block;
    int n = 0;
    for (uint32_t r = 0; r < kKv8Block; r++) n += b * kKv8Block + r >= start ? (int)c[r] - 128 : 0;
    sum += (double)n * (double)p.scales[2 * u + 1];
  }
  for (uint32_t r = start > own ? start - own : 0; r <= pos - own; r++) sum += (double)vo[r * vstride + d];
  return (float)(sum / (double)(pos + 1 - start));
}

struct Kv8Part {  // partial sums: o [part][n * n_heads][hd], then (max, sum) [part][n * n_heads]
  float* o;
  float2* ml;
};
__device__ __forceinline__ Kv8Part parts_of(const Kv8Args& a) {
  float* o = a.part;
  return {o, reinterpret_cast<float2*>(o + (size_t)a.nparts * a.n * a.n_heads * a.p.hd)};
}

// LDS of k8_rows in floats: queries, the own block's keys and values, its weights and sums, the waves' sums.
constexpr uint32_t kv8_pad(uint32_t hd) { return hd + 4; }
uint32_t kv8_rows_lds(uint32_t hd, uint32_t hdp, uint32_t rows) {
  return (16 * kv8_pad(hdp) + 2 * kKv8Block * kv8_pad(hd) + 16 * 16 + rows * kv8_pad(hd) + 4 * rows * kv8_pad(hdp)) * 4;
}

// STEP: group x is entry x, and the token is appended here. ONE: one workgroup takes both
// the own block and what is before it (at most kKv8Split positions), and writes the context.
template <int NS, bool STEP, bool ONE>
__global__ void __launch_bounds__(256, NS <= 6 ? 2 : 1) k8_rows(Kv8Args a, Kv8Inline inl) {
  constexpr uint32_t HDP = 32 * NS, NP = NS / 2, QS = kv8_pad(HDP);
  extern __shared__ float4 lds_v4[];
  __shared__ uint32_t red[8];
  __shared__ float own_m[16], own_l[16], wm[4][16], wl[4][16];
  const Kv8Pool& p = a.p;
  const uint32_t x = blockIdx.x, h = blockIdx.y, z = blockIdx.z, t = threadIdx.x, hd = p.hd, G = a.n_heads / p.n_kv;
  const uint32_t lane = t & 63, n16 = lane & 15, kg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  Kv8Run run;
  AttnEntry e{};
  if (STEP) {
    e = a.ent ? a.ent[x] : inl.e[x];
    run = Kv8Run{x, 1, e.pos, 0, (uint32_t)((e.pages - p.tables) / p.ppseq)};
  } else {
    run = a.run[x];
  }
  const uint32_t rows = run.n * G, hs = kv8_pad(hd);
  float* qs = reinterpret_cast<float*>(lds_v4);  // [16][QS]
  float* kt = qs + 16 * QS;                      // [16][hs], then the values
  float* vt = kt + kKv8Block * hs;
  float* ps = vt + kKv8Block * hs;               // [16][16]
  float* oo = ps + 16 * 16;                      // [rows][hs]
  float* wo = oo + rows * hs;                    // [4][rows][QS]
  auto start_of = [&](uint32_t pos) { return a.window && pos + 1 > a.window ? pos + 1 - a.window : 0; };
  const uint32_t own = run.pos0 / kKv8Block * kKv8Block, last = run.pos0 + run.n - 1;
  const uint32_t base = start_of(run.pos0) / kKv8Block * kKv8Block;
  const uint32_t lo = base + (ONE || z == 0 ? 0 : z - 1) * kKv8Split, hi = min(own, lo + kKv8Split);
  const Kv8Part part = parts_of(a);
  auto prow = [&](uint32_t r) {  // row r's place in a part
    return (size_t)z * a.n * a.n_heads + (size_t)(run.i0 + r / G) * a.n_heads + h * G + r % G;
  };
  if (!ONE && z && lo >= hi) {
    if (t < rows) part.ml[prow(t)] = make_float2(-INFINITY, 0.0f);
    return;
  }
  const bool mine = ONE || z == 0;
  // the first tile's codes on their way before the queries are turned
  const uint8_t *ka = nullptr, *va = nullptr;
  float sk = 0.0f, sv = 0.0f;
  uint4 kr[NP ? NP : 1][4], vr[2 * NS];
  uint2 kt8[4];
  auto find = [&](uint32_t kb) {  // this lane's addresses in the tile of four blocks at kb
    auto unit = [&](uint32_t j) {
      const uint32_t b = min(kb + kKv8Block * j, hi - 1) / kKv8Block;
      return kv8_block(p, kv8_page(p, run.table, b), b, h);
    };
    const size_t uk = unit(n16 / 4), uv = unit(kg);
    ka = p.codes + uk * (2 * kKv8Block * HDP) + (n16 % 4) * 64 + kg * 16;
    va = p.codes + uv * (2 * kKv8Block * HDP) + kKv8Block * HDP + n16 * kKv8Block;
    const float2 sc = reinterpret_cast<const float2*>(p.scales)[uv];
    sk = sc.x;
    sv = sc.y;
  };
  auto load_k = [&]() {
#pragma unroll
    for (int q = 0; q < 4; q++) {
#pragma unroll
      for (uint32_t u = 0; u < NP; u++) kr[u][q] = *reinterpret_cast<const uint4*>(ka + u * 1024 + q * 256);
      if (NS % 2)
        kt8[q] = *reinterpret_cast<const uint2*>(ka - (n16 % 4) * 64 - kg * 16 + NP * 1024 + (4 * q + n16 % 4) * 32 + kg * 8);
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int d = 0; d < 2 * NS; d++) vr[d] = *reinterpret_cast<const uint4*>(va + d * 256);
  };
  uint32_t kb = lo + 64 * wave;
  const bool any = (ONE || z) && kb < hi;
  if (any) {
    find(kb);
    load_k();
    load_v();
  }
  // queries, turned
  for (uint32_t y = t; y < rows * (HDP / 2); y += 256) {
    const uint32_t r = y / (HDP / 2), c = y % (HDP / 2);
    float2 w = make_float2(0.0f, 0.0f);
    if (2 * c < hd) {
      double cs, sn;
      turn(p.turns[c], run.pos0 + r / G, cs, sn);
      const float2 q = pair_of(a.q + (size_t)(run.i0 + r / G) * a.q_stride + (h * G + r % G) * hd, c, a.nsl, a.sl_stride);
      w = rotated(q.x, q.y, cs, sn);
    }
    reinterpret_cast<float2*>(qs + r * QS)[c] = w;
  }
  if (mine) {
    if (STEP) {
      const uint32_t block = run.pos0 / kKv8Block, r0 = run.pos0 % kKv8Block;
      if (e.fresh && h == 0 && t == 0) e.pages[run.pos0 / p.bs] = e.page;  // for the calls after this one
      block_rows(a, run.table, block, r0, 1, h, kt, vt, hs, [&](uint32_t) { return x; });
      __syncthreads();
      if (r0 == kKv8Block - 1) hold_block(p, kv8_block(p, e.page, block, h), kt, vt, hs, red);
      put_open(p, run.table, r0 + 1, h, kt, vt, hs);
    } else {
      const float* src = a.own + ((size_t)run.job * 2 * p.n_kv + h) * kKv8Block * hd;
      for (uint32_t y = t; y < kKv8Block * hd; y += 256) {
        kt[y / hd * hs + y % hd] = src[y];
        vt[y / hd * hs + y % hd] = src[(size_t)p.n_kv * kKv8Block * hd + y];
      }
    }
  }
  __syncthreads();
  const float sc2 = a.scale * kLog2e;
  if (mine) {
    // scores of (row, own position), several threads a dot; then softmax and P V in f32
    const uint32_t np = rows <= 4 ? 4 : rows <= 8 ? 2 : 1, pk = t / np, r = pk / 16, j = pk % 16;
    const uint32_t pr = run.pos0 + min(r, rows - 1) / G;
    if (r < rows) {
      float s = 0.0f;
      const float4 *q4 = reinterpret_cast<const float4*>(qs + r * QS), *k4 = reinterpret_cast<const float4*>(kt + j * hs);
      for (uint32_t d = t % np; d < hd / 4; d += np) {
        const float4 q = q4[d], k = k4[d];
        s = fmaf(q.x, k.x, s);
        s = fmaf(q.y, k.y, s);
        s = fmaf(q.z, k.z, s);
        s = fmaf(q.w, k.w, s);
      }
      for (uint32_t o = 1; o < np; o *= 2) s += __shfl_xor(s, o, 64);
      const bool in = own + j <= pr && own + j >= start_of(pr);
      s = in ? s * sc2 : -INFINITY;
      bool bad = s != s || s == INFINITY;
      float m = s;
      for (uint32_t o = np; o < 16 * np; o *= 2) {
        m = fmaxf(m, __shfl_xor(m, o, 64));
        bad |= __shfl_xor((int)bad, o, 64) != 0;
      }
      const float w = s > -INFINITY && !bad ? __builtin_amdgcn_exp2f(s - m) : 0.0f;
      float l = w;
      for (uint32_t o = np; o < 16 * np; o *= 2) l += __shfl_xor(l, o, 64);
      if (t % np == 0) ps[r * 16 + j] = w;
      if (t % np == 0 && j == 0) {
        own_m[r] = bad ? __uint_as_float(kBadRow) : m;
        own_l[r] = l;
      }
    }
    __syncthreads();
    for (uint32_t y = t; y < rows * hd; y += 256) {
      const uint32_t r = y / hd, d = y % hd, pr = run.pos0 + r / G, st = start_of(pr);
      float o = 0.0f;
      for (uint32_t j = st > own ? st - own : 0; j <= pr - own; j++) o = fmaf(ps[r * 16 + j], vt[j * hs + d], o);
      if (ONE) oo[r * hs + d] = o;
      else part.o[prow(r) * hd + d] = o;
    }
    if (!ONE) {
      if (t < rows) part.ml[prow(t)] = make_float2(own_m[t], own_l[t]);
      return;
    }
  }
  // B operand of the queries: the lane's column is row n16
  f16x8 qh[NS], ql[NS];
  float cq;
  bool bad;
  {
    const uint32_t r = min(n16, rows - 1);
    float4 v[NS][2];
    float m = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const uint32_t d = NS % 2 && s == NS - 1 ? 64 * NP + 8 * kg : 64 * (s / 2) + 16 * kg + 8 * (s % 2);
#pragma unroll
      for (int y = 0; y < 2; y++) {
        v[s][y] = reinterpret_cast<const float4*>(qs + r * QS + d)[y];
        for (float f : {v[s][y].x, v[s][y].y, v[s][y].z, v[s][y].w}) {
          m = fmaxf(m, fabsf(f));
          top = max(top, __float_as_uint(f) & 0x7fffffffu);
        }
      }
    }
    m = max16_32(m);
    bad = max16_32(top >= 0x7f800000u ? 1.0f : 0.0f) != 0.0f;
    const int eq = bad ? 0 : pow2_of(m);
    const float up = bad ? 0.0f : pow2(9 - eq);  // the largest in [2^9, 2^10): what is left of it is no denormal
    cq = sc2 * pow2(max(eq - 9, -126));
#pragma unroll
    for (int s = 0; s < NS; s++) {
      float f[8];
#pragma unroll
      for (int y = 0; y < 2; y++) {
        f[4 * y] = v[s][y].x * up;
        f[4 * y + 1] = v[s][y].y * up;
        f[4 * y + 2] = v[s][y].z * up;
        f[4 * y + 3] = v[s][y].w * up;
      }
      if (bad)
        for (int y = 0; y < 8; y++) f[y] = 0.0f;
      split8(f, qh[s], ql[s]);
    }
  }
  const uint32_t pos_n = run.pos0 + min(n16, rows - 1) / G, start_n = start_of(pos_n);
  const uint32_t start_max = start_of(last);
  f32x4 o[2 * NS];
#pragma unroll
  for (int d = 0; d < 2 * NS; d++) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float M = -INFINITY, L = 0.0f;
  int ev = -100;  // the values' sums are in units of 2^ev, at least the largest scale's
  if (any)
    for (;;) {
      f32x4 s[4];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        s[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NS; c++) {
          uint32_t w0, w1;
          if (NS % 2 && c == NS - 1) {
            w0 = kt8[q].x;
            w1 = kt8[q].y;
          } else {
            const uint4 k = kr[c / 2][q];
            w0 = c % 2 ? k.z : k.x;
            w1 = c % 2 ? k.w : k.y;
          }
          const f16x8 kf = codes8(w0, w1);
          s[q] = mfma16(kf, ql[c], s[q]);
          s[q] = mfma16(kf, qh[c], s[q]);
        }
      }
      const float ck = sk * cq, svn0 = sv;
      const uint32_t k0 = kb + kKv8Block * kg;
      const bool edge = kb < start_max || kb + 64 > hi;  // the same in every lane
      kb += 256;
      const bool more = kb < hi;
      if (more) {
        find(kb);
        load_k();
      }
      float svn = svn0;
#pragma unroll
      for (int q = 0; q < 4; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[q][r] *= ck;
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const uint32_t pk = k0 + 4 * q + r;
            if (pk < start_n || pk >= hi) s[q][r] = -INFINITY;
          }
        if (k0 >= hi || k0 + kKv8Block <= start_n) svn = 0.0f;  // no position of the block is attended to
      }
      float mt = -INFINITY;
#pragma unroll
      for (int q = 0; q < 4; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          bad |= __builtin_amdgcn_classf(s[q][r], 0x203);  // NaN or +inf
          mt = fmaxf(mt, s[q][r]);
        }
      mt = fmaxf(M, max16_32(mt) - 14.0f);
      const int en = max(ev, (int)max16_32((float)pow2_of(svn)));
      // weights are 2^(s - M), at most 2^14: M is the largest score less 14
      const float mu = mt == -INFINITY ? 0.0f : mt;
      float f = __builtin_amdgcn_exp2f(M - mu);
      L *= f;
      f *= pow2(max(ev - en, -126));
      if (__ballot(f != 1.0f)) {
#pragma unroll
        for (int d = 0; d < 2 * NS; d++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[d][r] *= f;
      }
      M = mt;
      ev = en;
      const float vn = svn * pow2(-en);  // below 2: weights up to 2^15
      f16x8 wh[2], wl2[2];
#pragma unroll
      for (int y = 0; y < 2; y++) {
        float w[8];
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float pv = __builtin_amdgcn_exp2f(s[2 * y + q][r] - mu);
            L += pv;
            w[4 * q + r] = pv * vn;
          }
        split8(w, wh[y], wl2[y]);
      }
#pragma unroll
      for (int d = 0; d < 2 * NS; d++) {
        const uint4 v = vr[d];
        const f16x8 v0 = codes8(v.x, v.y), v1 = codes8(v.z, v.w);
        o[d] = mfma16(v0, wl2[0], o[d]);
        o[d] = mfma16(v1, wl2[1], o[d]);
        o[d] = mfma16(v0, wh[0], o[d]);
        o[d] = mfma16(v1, wh[1], o[d]);
      }
      if (!more) break;
      load_v();
    }
  // the waves' sums joined through LDS, the values' in natural units
  L = sum16_32(L);
  bad = max16_32(bad ? 1.0f : 0.0f) != 0.0f;
  const float fo = pow2(ev);
  if (n16 < rows) {
    if (kg == 0) {
      wm[wave][n16] = bad ? __uint_as_float(kBadRow) : M;
      wl[wave][n16] = L;
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; d++)
      *reinterpret_cast<float4*>(wo + (wave * rows + n16) * QS + 16 * d + 4 * kg) =
          make_float4(o[d][0] * fo, o[d][1] * fo, o[d][2] * fo, o[d][3] * fo);
  }
  __syncthreads();
  for (uint32_t y = t; y < rows * hd; y += 256) {
    const uint32_t r = y / hd, d = y % hd;
    float m = -INFINITY, l = 0.0f, v = 0.0f;
    bool bd = false;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      bd |= wm[w][r] != wm[w][r];
      m = fmaxf(m, wm[w][r]);
    }
    if (m > -INFINITY)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        if (!(wm[w][r] > -INFINITY)) continue;
        const float f = __builtin_amdgcn_exp2f(wm[w][r] - m);
        l += wl[w][r] * f;
        v += wo[(w * rows + r) * QS + d] * f;
      }
    if (bd) m = __uint_as_float(kBadRow);
    if (!ONE) {
      part.o[prow(r) * hd + d] = v;
      if (d == 0) part.ml[prow(r)] = make_float2(m, l);
      continue;
    }
    // the own block's part and this one, as k8_join joins parts
    const float m0 = own_m[r], mm = fmaxf(m0, m);
    const uint32_t pr = run.pos0 + r / G;
    float c;
    if (bd || m0 != m0 || mm == -INFINITY) {
      c = uniform_mean(p, run.table, h, start_of(pr), pr, d, vt, hs);
    } else {
      float la = 0.0f, oa = 0.0f, lb = 0.0f, ob = 0.0f;
      if (m0 > -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(m0 - mm);
        la += own_l[r] * f;
        oa += oo[r * hs + d] * f;
      }
      if (m > -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(m - mm);
        lb += l * f;
        ob += v * f;
      }
      c = (oa + ob) / (la + lb);
    }
    a.ctx[((size_t)(run.i0 + r / G) * a.n_heads + h * G + r % G) * hd + d] = c;
  }
}

// grid (n, n_heads), 256 threads: a row's parts joined, threads of several groups taking
// every ng-th part for four columns each, the groups then added in order.
template <bool STEP>
__global__ void __launch_bounds__(256) k8_join(Kv8Args a, Kv8Inline inl) {
  __shared__ float4 go[256];
  __shared__ float gl[256], gm[4];
  const Kv8Pool& p = a.p;
  const uint32_t i = blockIdx.x, hh = blockIdx.y, t = threadIdx.x, hd = p.hd, q4 = hd / 4, ng = 256 / q4, g = t / q4, c = t % q4;
  const size_t rows = (size_t)a.n * a.n_heads, row = (size_t)i * a.n_heads + hh;
  const Kv8Part part = parts_of(a);
  float m = -INFINITY;
  bool bad = false;
  for (uint32_t s = t; s < a.nparts; s += 256) {
    const float v = part.ml[s * rows + row].x;
    bad |= v != v;
    m = fmaxf(m, v);
  }
  m = wave64_max(m);
  if (__ballot(bad)) m = INFINITY;  // no part's maximum is: the mark
  if ((t & 63) == 0) gm[t >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
  const bool uniform = m == INFINITY || m == -INFINITY;
  float l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (g < ng && !uniform)
    for (uint32_t s0 = g; s0 < a.nparts; s0 += 4 * ng) {
      float2 v[4];
      float4 w[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; k++) {
        const uint32_t s = s0 + k * ng;
        v[k] = make_float2(-INFINITY, 0.0f);
        if (s < a.nparts) {
          v[k] = part.ml[s * rows + row];
          w[k] = reinterpret_cast<const float4*>(part.o + (s * rows + row) * hd)[c];
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; k++) {
        if (!(v[k].x > -INFINITY)) continue;
        const float f = __builtin_amdgcn_exp2f(v[k].x - m);
        l += v[k].y * f;
        o = make_float4(o.x + w[k].x * f, o.y + w[k].y * f, o.z + w[k].z * f, o.w + w[k].w * f);
      }
    }
  go[t] = o;
  gl[t] = l;
  __syncthreads();
  if (t >= q4) return;
  if (!uniform) {
    for (uint32_t k = 1; k < ng; k++) {
      const float4 b = go[k * q4 + t];
      l += gl[k * q4 + t];
      o = make_float4(o.x + b.x, o.y + b.y, o.z + b.z, o.w + b.w);
    }
    o = make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
  } else {
    const uint32_t h = hh / (a.n_heads / p.n_kv);
    uint32_t pos, table;
    const float* vo;
    if (STEP) {
      const AttnEntry e = a.ent ? a.ent[i] : inl.e[i];
      pos = e.pos;
      table = (uint32_t)((e.pages - p.tables) / p.ppseq);
      vo = kv8_open(p, table, h) + (size_t)p.n_kv * kKv8Block * hd;
    } else {
      uint32_t r = 0;
      while (i - a.run[r].i0 >= a.run[r].n) r++;
      const Kv8Run run = a.run[r];
      pos = run.pos0 + i - run.i0;
      table = run.table;
      vo = a.own + (((size_t)run.job * 2 + 1) * p.n_kv + h) * kKv8Block * hd;
    }
    const uint32_t start = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
    float u[4];
    for (uint32_t k = 0; k < 4; k++) u[k] = uniform_mean(p, table, h, start, pos, 4 * t + k, vo, hd);
    o = make_float4(u[0], u[1], u[2], u[3]);
  }
  float* dst = a.ctx + row * hd + 4 * t;
  dst[0] = o.x;
  dst[1] = o.y;
  dst[2] = o.z;
  dst[3] = o.w;
}

// grid (chunks, n_kv), 256 threads: rows of one block, from its codes or from the open rows.
__global__ void __launch_bounds__(256) k8_read(Kv8Pool p, const Kv8Rows* rows, Kv8RowsInline inl, float* k, float* v) {
  const Kv8Rows r = rows ? rows[blockIdx.x] : inl.r[blockIdx.x];
  const uint32_t h = blockIdx.y, hd = p.hd, kvd = p.n_kv * hd;
  float* dk = k + (size_t)r.i0 * kvd + h * hd;
  float* dv = v + (size_t)r.i0 * kvd + h * hd;
  if (!r.whole) {
    const float* src = kv8_open(p, r.table, h) + r.r0 * hd;
    for (uint32_t x = threadIdx.x; x < r.n * hd; x += 256) {
      const size_t to = (size_t)(x / hd) * kvd + x % hd;
      dk[to] = src[x];
      dv[to] = src[(size_t)p.n_kv * kKv8Block * hd + x];
    }
    return;
  }
  const size_t u = kv8_block(p, kv8_page(p, r.table, r.block), r.block, h);
  const uint8_t* c = kv8_codes(p, u);
  const float sk = p.scales[2 * u], sv = p.scales[2 * u + 1];
  for (uint32_t x = threadIdx.x; x < r.n * hd; x += 256) {
    const uint32_t row = r.r0 + x / hd, d = x % hd;
    const size_t to = (size_t)(x / hd) * kvd + d;
    dk[to] = (float)((int)c[kv8_key(p.hdp, row, d)] - 128) * sk;
    dv[to] = (float)((int)c[kKv8Block * p.hdp + d * kKv8Block + row] - 128) * sv;
  }
}

// grid (blocks, n_kv), 256 threads: rows r0 .. r0 + n - 1 of a held block become open rows.
__global__ void __launch_bounds__(256) k8_reopen(Kv8Pool p, Kv8RowsInline inl) {
  const Kv8Rows r = inl.r[blockIdx.x];
  const uint32_t h = blockIdx.y, hd = p.hd;
  const size_t u = kv8_block(p, kv8_page(p, r.table, r.block), r.block, h);
  const uint8_t* c = kv8_codes(p, u);
  const float sk = p.scales[2 * u], sv = p.scales[2 * u + 1];
  float* to = kv8_open(p, r.table, h) + r.r0 * hd;
  for (uint32_t x = threadIdx.x; x < r.n * hd; x += 256) {
    const uint32_t row = r.r0 + x / hd, d = x % hd;
    to[x] = (float)((int)c[kv8_key(p.hdp, row, d)] - 128) * sk;
    to[(size_t)p.n_kv * kKv8Block * hd + x] = (float)((int)c[kKv8Block * p.hdp + d * kKv8Block + row] - 128) * sv;
  }
}

bool overlaps(const float* a, size_t na, const float* b, size_t nb) { return a < b + nb && b < a + na; }

// One workgroup a group and kv head: everything before the own block fits one part, and no
// other workgroup's input lies under the context.
bool one_part(const Kv8Args& a, bool step) {
  const size_t n = a.n, qd = (size_t)a.n_heads * a.p.hd, kvd = (size_t)a.p.n_kv * a.p.hd;
  const size_t more = a.nsl > 1 ? (a.nsl - 1) * a.sl_stride : 0;
  auto over = [&](const float* p, size_t width, size_t stride) {
    return overlaps(a.ctx, n * qd, p, (n - 1) * stride + width + more);
  };
  if (a.nparts != 2 || over(a.q, qd, a.q_stride)) return false;
  return !step || (!over(a.k, kvd, a.kv_stride) && !over(a.v, kvd, a.kv_stride));
}

template <int NS, bool STEP>
void launch_rows(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) {
  const bool one = one_part(a, STEP);
  // what 16 rows of the widest heads of this build take, set once; a call asks for its own rows'
  static const bool set = [] {
    const int most = (int)kv8_rows_lds(32 * NS, 32 * NS, 16);
    return hipFuncSetAttribute((const void*)k8_rows<NS, STEP, true>, hipFuncAttributeMaxDynamicSharedMemorySize, most) == hipSuccess &&
           hipFuncSetAttribute((const void*)k8_rows<NS, STEP, false>, hipFuncAttributeMaxDynamicSharedMemorySize, most) == hipSuccess;
  }();
  (void)set;
  const uint32_t G = a.n_heads / a.p.n_kv, rows = STEP ? G : kv8_group_tokens(G) * G;
  const uint32_t lds = kv8_rows_lds(a.p.hd, a.p.hdp, rows);
  const dim3 grid(STEP ? a.n : a.nrun, a.p.n_kv, one ? 1 : a.nparts);
  auto kernel = one ? k8_rows<NS, STEP, true> : k8_rows<NS, STEP, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, a, inl);
  if (!one) hipLaunchKernelGGL(k8_join<STEP>, dim3(a.n, a.n_heads), dim3(256), 0, st, a, inl);
}

template <bool STEP>
hipError_t launch_rows_of(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) {
  switch (a.p.hdp / 32) {
    case 1: launch_rows<1, STEP>(a, inl, st); break;
    case 2: launch_rows<2, STEP>(a, inl, st); break;
    case 3: launch_rows<3, STEP>(a, inl, st); break;
    case 4: launch_rows<4, STEP>(a, inl, st); break;
    case 6: launch_rows<6, STEP>(a, inl, st); break;
    default: launch_rows<8, STEP>(a, inl, st); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_step(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) { return launch_rows_of<true>(a, inl, st); }

hipError_t launch_kv8_call(const Kv8Args& a, hipStream_t st) {
  hipLaunchKernelGGL(k8_append, dim3(a.njob, a.p.n_kv), dim3(256), 2 * kKv8Block * a.p.hd * 4, st, a);
  if (!a.ctx) return hipGetLastError();
  return launch_rows_of<false>(a, Kv8Inline{}, st);
}

hipError_t launch_kv8_read(const Kv8Pool& p, const Kv8Rows* rows, const Kv8RowsInline& inl, uint32_t nrows, float* k,
                           float* v, hipStream_t st) {
  hipLaunchKernelGGL(k8_read, dim3(nrows, p.n_kv), dim3(256), 0, st, p, rows, inl, k, v);
  return hipGetLastError();
}

hipError_t launch_kv8_reopen(const Kv8Pool& p, const Kv8RowsInline& inl, uint32_t nrows, hipStream_t st) {
  hipLaunchKernelGGL(k8_reopen, dim3(nrows, p.n_kv), dim3(256), 0, st, p, inl);
  return hipGetLastError();
}

}  // namespace gmoe
