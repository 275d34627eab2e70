// gmoe_attn8.hip — the paged KV cache held in 8 bits: append, attention, reading back.
//
// A sequence's positions are cut into blocks of 16. Of a complete block, one kv head's keys
// (values) x are held as codes c = rint(x * (127 * (1 / m))), m = max |x| over the block's 16
// rows, and a scale s = m / 127 rounded to f32; they stand for c * s. The block of the sequence's
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

#include <type_traits>

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

constexpr uint32_t kv8_pad(uint32_t hd) { return hd + 4; }  // floats between rows in LDS: 16 rows' columns on all banks

__device__ __forceinline__ void turn(double turns, uint32_t pos, double& c, double& s) {
  double t = (double)pos * turns;
  t -= rint(t);
  sincospi(2.0 * t, &s, &c);
}
__device__ __forceinline__ float2 rotated(float x, float y, double c, double s) {
  const double a = x, b = y;
  return make_float2((float)(a * c - b * s), (float)(a * s + b * c));
}

// Whether this workgroup is the last of `n` to have written its part: the others' are then in
// memory. Every thread calls it; `last` is a word of LDS. The last one sets the counter back for
// the next call on the cache. Parts are written and read by accesses of device scope, which
// go past the XCDs' own caches, so that all that is waited for is the workgroup's own stores (a fence of
// that scope writes a whole cache back for every wave: 8 sequences at 65000 in 1630 us).
__device__ __forceinline__ bool last_part(uint32_t* done, uint32_t n, uint32_t* last) {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    *last = atomicAdd(done, 1u) == n - 1 ? 1u : 0u;
    if (*last) *done = 0;
  }
  __syncthreads();
  return *last != 0;
}
__device__ __forceinline__ void store_shared2(float* p, float2 v) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared2(const float* p) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void store_shared4(float* p, float4 v) {
  store_shared2(p, make_float2(v.x, v.y));
  store_shared2(p + 2, make_float2(v.z, v.w));
}
__device__ __forceinline__ float4 load_shared4(const float* p) {
  const float2 a = load_shared2(p), b = load_shared2(p + 2);
  return make_float4(a.x, a.y, b.x, b.y);
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows of the caller's: any float's alignment
__device__ __forceinline__ float4 load4(const float* p) {
  const f32x4u v = *reinterpret_cast<const f32x4u*>(p);
  return make_float4(v.x, v.y, v.z, v.w);
}
// Four elements from p on: sums of nsl slices in slice order.
__device__ __forceinline__ float4 four_of(const float* p, uint32_t nsl, uint64_t stride) {
  float4 v = load4(p);
  for (uint32_t g = 1; g < nsl; g++) {
    const float4 w = load4(p + g * stride);
    v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
  }
  return v;
}
// Elements 4c .. 4c + 3 of a head's row at position pos, turned.
__device__ __forceinline__ float4 turned(const Kv8Pool& p, float4 v, uint32_t c, uint32_t pos) {
  double cs[2], sn[2];
  for (uint32_t i = 0; i < 2; i++) turn(p.turns[2 * c + i], pos, cs[i], sn[i]);
  const float2 a = rotated(v.x, v.y, cs[0], sn[0]), b = rotated(v.z, v.w, cs[1], sn[1]);
  return make_float4(a.x, a.y, b.x, b.y);
}

// The rows of one block and kv head in a thread's registers, 256 threads: float4 i of the keys'
// [16][HDP] then the values', i = t + 256 y. All loads are in flight together (one after another they
// were most of a short call).
template <int NS>
struct BlockRows {
  static constexpr uint32_t Q4 = 8 * NS;  // float4 of a row
  float4 v[NS];
  static __device__ uint32_t value(uint32_t i) { return i / (16 * Q4); }
  static __device__ uint32_t row(uint32_t i) { return i / Q4 % 16; }
  static __device__ uint32_t col(uint32_t i) { return i % Q4; }

  // Rows below r0 from the open rows, the next n from k and v (keys not yet turned), row r being
  // entry ent(r); zeros after them and past the head's width.
  template <class F>
  __device__ __forceinline__ void load(const Kv8Args& a, uint32_t table, uint32_t r0, uint32_t n, uint32_t h, F&& ent) {
    const Kv8Pool& p = a.p;
    const float* old = kv8_open(p, table, h);
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      const uint32_t i = threadIdx.x + 256 * y, r = row(i), c = col(i);
      v[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (4 * c >= p.hd || r >= r0 + n) continue;
      if (r < r0) v[y] = *reinterpret_cast<const float4*>(old + (size_t)value(i) * p.n_kv * kKv8Block * p.hd + r * p.hd + 4 * c);
      else v[y] = four_of((value(i) ? a.v : a.k) + (size_t)ent(r) * a.kv_stride + h * p.hd + 4 * c, a.nsl, a.sl_stride);
    }
  }
  __device__ __forceinline__ void turn_keys(const Kv8Pool& p, uint32_t block, uint32_t r0, uint32_t n) {
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      const uint32_t i = threadIdx.x + 256 * y, r = row(i), c = col(i);
      if (!value(i) && 4 * c < p.hd && r >= r0 && r < r0 + n) v[y] = turned(p, v[y], c, block * kKv8Block + r);
    }
  }
  // to LDS, rows hs floats apart (hs at least HDP)
  __device__ __forceinline__ void put(float* kt, float* vt, uint32_t hs) const {
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      const uint32_t i = threadIdx.x + 256 * y;
      *reinterpret_cast<float4*>((value(i) ? vt : kt) + row(i) * hs + 4 * col(i)) = v[y];
    }
  }
  // the first n rows to [2][n_kv][16][hd] at to (of kv head 0); SHARED: for other workgroups of the launch
  template <bool SHARED = false>
  __device__ __forceinline__ void put_global(const Kv8Pool& p, float* to, uint32_t h, uint32_t n) const {
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      const uint32_t i = threadIdx.x + 256 * y, r = row(i), c = col(i);
      if (r >= n || 4 * c >= p.hd) continue;
      float* d = to + (((size_t)value(i) * p.n_kv + h) * kKv8Block + r) * p.hd + 4 * c;
      if (SHARED) store_shared4(d, v[y]);
      else *reinterpret_cast<float4*>(d) = v[y];
    }
  }
  // the largest magnitudes of keys and values, as bits: a NaN's above infinity's above every
  // number's. red: 8 words of LDS.
  __device__ __forceinline__ uint2 largest(uint32_t* red) const {
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      uint32_t m = 0;
      for (float f : {v[y].x, v[y].y, v[y].z, v[y].w}) m = max(m, __float_as_uint(f) & 0x7fffffffu);
      if (value(threadIdx.x + 256 * y)) mv = max(mv, m);
      else mk = max(mk, m);
    }
    for (int o = 32; o; o >>= 1) {
      mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
      mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
    }
    const uint32_t t = threadIdx.x;
    if ((t & 63) == 0) {
      red[t >> 6] = mk;
      red[4 + (t >> 6)] = mv;
    }
    __syncthreads();
    return make_uint2(max(max(red[0], red[1]), max(red[2], red[3])), max(max(red[4], red[5]), max(red[6], red[7])));
  }
};

// A block's 16 rows (in LDS, hs floats apart), of largest magnitudes m, to codes and scales.
template <int NS>
__device__ __forceinline__ void hold_block(const Kv8Pool& p, size_t unit, const float* kt, const float* vt, uint32_t hs, uint2 m) {
  constexpr uint32_t HDP = 32 * NS, W = kKv8Block * HDP / 4;  // words of the keys', and of the values' codes
  const uint32_t t = threadIdx.x;
  // 127 times 1 / m, as a program without a kernel forms it: on a tie (x = m / 2) the product's last
  // bit decides, and the same operations give the same code
  auto inv = [](uint32_t m) { return m == 0 || m >= 0x7f800000u ? 0.0 : 127.0 * (1.0 / (double)__uint_as_float(m)); };
  auto scale = [](uint32_t m) {
    return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (float)((double)__uint_as_float(m) / 127.0);
  };
  // a NaN's code is any: its block's scale says so
  auto code = [](float x, double i) { return i == 0.0 ? 128u : (uint32_t)((int)rint((double)x * i) + 128) & 255u; };
  const double ik = inv(m.x), iv = inv(m.y);
  uint8_t* dst = kv8_codes(p, unit);
#pragma unroll
  for (uint32_t y = 0; y < W; y += 256) {
    const uint32_t x = y + t, r = x / (HDP / 4), d = x % (HDP / 4) * 4;
    if (W % 256 && x >= W) break;
    uint32_t w = 0;
#pragma unroll
    for (uint32_t b = 0; b < 4; b++) w |= code(kt[r * hs + d + b], ik) << 8 * b;  // zeros past the head's width
    *reinterpret_cast<uint32_t*>(dst + kv8_key(HDP, r, d)) = w;
  }
  uint32_t* vd = reinterpret_cast<uint32_t*>(dst + kKv8Block * HDP);
#pragma unroll
  for (uint32_t y = 0; y < W; y += 256) {
    const uint32_t x = y + t, d = x / 4, r = x % 4 * 4;
    if (W % 256 && x >= W) break;
    uint32_t w = 0;
#pragma unroll
    for (uint32_t b = 0; b < 4; b++) w |= code(vt[(r + b) * hs + d], iv) << 8 * b;
    vd[x] = w;
  }
  if (t == 0) {
    p.scales[2 * unit] = scale(m.x);
    p.scales[2 * unit + 1] = scale(m.y);
  }
}

// grid (njob * n_kv, 1, 1 + ceil(G / 4) where the call attends), 256 threads: a block of the call's
// positions and one kv head's keys and values (z 0), or up to four of its query heads, whose
// turned rows go to a.qr. The job of a sequence's first block writes the open rows of its last
// one, after it has read those that were there. Copies the call's groups and tiles to the
// device for the launches after it.
// I: Kv8CallInline, or without one OfHost (3 kB of arguments cost the host 0.5 us).
struct OfHost {};
template <int NS, class I>
__global__ void __launch_bounds__(256) k8_append(Kv8Args a, I inl) {
  constexpr bool INL = std::is_same<I, Kv8CallInline>::value;
  constexpr uint32_t HS = kv8_pad(32 * NS), Q4 = 8 * NS;
  __shared__ __attribute__((aligned(16))) float kt[kKv8Block * HS], vt[kKv8Block * HS];
  __shared__ uint32_t red[8];
  __shared__ Kv8Job job;
  const Kv8Pool& p = a.p;
  const uint32_t h = blockIdx.x % p.n_kv, jb = blockIdx.x / p.n_kv, t = threadIdx.x;
  auto take = [&](uint32_t i) {  // job i
    auto word = [&](const Kv8Job* j) { return reinterpret_cast<const uint32_t*>(j + i)[t]; };
    if (t < sizeof(Kv8Job) / 4) {
      if constexpr (INL) reinterpret_cast<uint32_t*>(&job)[t] = word(inl.j);
      else reinterpret_cast<uint32_t*>(&job)[t] = word(a.hjob);
    }
    __syncthreads();
  };
  take(jb);
  if (blockIdx.z) {
    const uint32_t G = a.n_heads / p.n_kv, g0 = 4 * (blockIdx.z - 1), ng = min(G - g0, 4u);
    float4 q[2 * NS];  // float4 t + 256 y of [ng][16][HDP], in flight together
    auto at = [&](uint32_t y, uint32_t& g, uint32_t& r, uint32_t& c) {
      const uint32_t i = t + 256 * y;
      c = i % Q4;
      r = i / Q4 % 16;
      g = i / Q4 / 16;
      return g < ng && r >= job.r0 && r < job.r0 + job.n && 4 * c < p.hd;
    };
#pragma unroll
    for (uint32_t y = 0; y < 2 * NS; y++) {
      uint32_t g, r, c;
      if (at(y, g, r, c)) q[y] = load4(a.q + (size_t)job.ent[r] * a.q_stride + (h * G + g0 + g) * p.hd + 4 * c);
    }
    // a thread's floats of one row and column in several heads share their angles
#pragma unroll
    for (uint32_t y = 0; y < 2 * NS; y++) {
      uint32_t g, r, c;
      if (at(y, g, r, c))
        *reinterpret_cast<float4*>(a.qr + ((size_t)job.ent[r] * a.n_heads + h * G + g0 + g) * p.hd + 4 * c) =
            turned(p, q[y], c, job.block * kKv8Block + r);
    }
    return;
  }
  const uint32_t flags = job.flags, last = job.last;
  if (h == 0 && t == 0 && (flags & kKv8Fresh))
    p.tables[(size_t)job.table * p.ppseq + job.block / (p.bs / kKv8Block)] = job.page;
  if (h == 0 && a.qr)
    for (uint32_t x = jb * 256 + t; x < a.nrun + a.ntile; x += a.njob * 256) {
      if constexpr (INL) a.run[x] = inl.r[x];
      else a.run[x] = a.hrun[x];
    }
  BlockRows<NS> rows;
  auto get = [&] {
    rows.load(a, job.table, job.r0, job.n, h, [&](uint32_t r) { return job.ent[r]; });
    rows.turn_keys(p, job.block, job.r0, job.n);
  };
  get();
  if (a.qr || (flags & kKv8Whole)) {
    const uint2 m = rows.largest(red);
    if (a.qr) {
      rows.put_global(p, a.own + (size_t)jb * 2 * p.n_kv * kKv8Block * p.hd, h, kKv8Block);
      if (t == 0) a.own_max[(size_t)jb * p.n_kv + h] = make_float2(__uint_as_float(m.x), __uint_as_float(m.y));
    }
    if (flags & kKv8Whole) {
      rows.put(kt, vt, HS);
      __syncthreads();
      hold_block<NS>(p, kv8_block(p, job.page, job.block, h), kt, vt, HS, m);
    }
  }
  if (!(flags & kKv8First)) return;
  if (last != jb) {
    __syncthreads();
    take(last);
    get();
  }
  rows.put_global(p, p.open + (size_t)job.table * 2 * p.n_kv * kKv8Block * p.hd, h, job.r0 + job.n);
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
// Codes go from memory to registers as the MFMAs want them, no LDS on the way. The last
// workgroup of a group to finish joins its parts, in their order, so a row's bits depend neither
// on the batch nor on how the workgroups were scheduled.
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
// Two values as two fp16 each: the first to nearest, the second what it leaves, truncated (within
// 2^-21 of the value, of either sign). The value is made opaque first: a product's conversion may be
// folded into one instruction that rounds the product once, and what is left of the product's
// f32 value then belongs to another first half. `one` is 1, opaque too, so that the subtraction
// is a v_fma_mix_f32, which takes the half as it stands.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  float one = 1.0f;
  asm("" : "+v"(x), "+v"(y), "+s"(one));
  const f16x2 h = __builtin_convertvector((f32x2{x, y}), f16x2);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h[0], -one, x),
                                                               __builtin_fmaf((float)h[1], -one, y)));
}
__device__ __forceinline__ void split8(const float* x, f16x8& hi, f16x8& lo) {
  u32x4 h, l;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t a, b;
    split2(x[2 * i], x[2 * i + 1], a, b);
    h[i] = a;
    l[i] = b;
  }
  hi = __builtin_bit_cast(f16x8, h);
  lo = __builtin_bit_cast(f16x8, l);
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

// A score's scale where the block's is 0, as its products are: for masked ones, -inf, to stay that.
__device__ __forceinline__ float above0(float x) { return x == 0.0f ? 1.0f : x; }

constexpr float kLog2e = 0x1.715476p+0f;
constexpr uint32_t kBadRow = 0x7fc00000u;  // a part's maximum: a NaN or +inf score

// A row's mean over its span, column d: uniform weights (rare). vo: its own block's values.
__device__ float uniform_mean(const Kv8Pool& p, uint32_t table, uint32_t h, uint32_t start, uint32_t pos, uint32_t d,
                              const float* vo, uint32_t vstride, bool shared = false) {
  const uint32_t own = pos / kKv8Block * kKv8Block;
  double sum = 0.0;
  for (uint32_t b = start / kKv8Block; b * kKv8Block < own; b++) {
    const size_t u = kv8_block(p, kv8_page(p, table, b), b, h);
    const uint8_t* c = kv8_codes(p, u) + kKv8Block * p.hdp + d * kKv8Block;
    int n = 0;
    for (uint32_t r = 0; r < kKv8Block; r++) n += b * kKv8Block + r >= start ? (int)c[r] - 128 : 0;
    sum += (double)n * (double)p.scales[2 * u + 1];
  }
  for (uint32_t r = start > own ? start - own : 0; r <= pos - own; r++) {
    const float* v = vo + r * vstride + d;
    sum += (double)(shared ? __hip_atomic_load(v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *v);
  }
  return (float)(sum / (double)(pos + 1 - start));
}

// Partial sums of the rows of nx groups (or tiles), up to R a kv head: o [part][group][kv head]
// [R][hd], then (max, sum) [part][group][kv head][R].
struct Kv8Part {
  float* o;
  float2* ml;
  uint32_t nx, n_kv, R;
  __device__ size_t row(uint32_t z, uint32_t x, uint32_t h, uint32_t r) const {
    return (((size_t)z * nx + x) * n_kv + h) * R + r;
  }
};
__device__ __forceinline__ Kv8Part parts_of(const Kv8Args& a, float* o, uint32_t nparts, uint32_t nx, uint32_t R) {
  return {o, reinterpret_cast<float2*>(o + (size_t)nparts * nx * a.p.n_kv * R * a.p.hd), nx, a.p.n_kv, R};
}
// First position that a token attends to.
__device__ __forceinline__ uint32_t kv8_start(const Kv8Args& a, uint32_t pos) {
  return a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
}
__device__ __forceinline__ Kv8Part rows_parts(const Kv8Args& a, bool step) {
  const uint32_t G = a.n_heads / a.p.n_kv;
  return parts_of(a, a.part, a.nparts, step ? a.n : a.nrun, step ? G : kv8_group_tokens(G) * G);
}

// Sums of one row's four columns over parts: o and l in units of 2^m. A part's sums come times the
// power that takes its maximum to the largest, rounded, then added; ok turns false at a maximum that
// is a NaN.
struct Joined {
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -INFINITY, l = 0.0f;
  bool ok = true;
  __device__ __forceinline__ void raise(float to) {
    if (!(to > m)) return;
    const float f = __builtin_amdgcn_exp2f(m - to);
    l *= f;
    o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    m = to;
  }
  __device__ __forceinline__ void add(float pm, float pl, const float4& p) {  // pm at most m
    if (!(pm > -INFINITY)) return;  // a part without a score: its sums may be unwritten
    const float f = __builtin_amdgcn_exp2f(pm - m);
    l += pl * f;
    o = make_float4(o.x + p.x * f, o.y + p.y * f, o.z + p.z * f, o.w + p.w * f);
  }
  // parts s0 .. s1 - 1 in order, N of them loaded at a time. SHARED: from workgroups of this launch.
  template <bool SHARED, uint32_t N>
  __device__ __forceinline__ void parts(const Kv8Part& part, uint32_t s0, uint32_t s1, size_t row, uint32_t hd, uint32_t c) {
    const size_t step = part.row(1, 0, 0, 0);
    for (; s0 < s1; s0 += N) {
      float2 v[N];
      float4 w[N];
      float mb = m;
#pragma unroll
      for (uint32_t k = 0; k < N; k++) {
        v[k] = make_float2(-INFINITY, 0.0f);
        if (s0 + k < s1) {
          const float2* ml = part.ml + (s0 + k) * step + row;
          const float* po = part.o + ((s0 + k) * step + row) * hd + 4 * c;
          v[k] = SHARED ? load_shared2(reinterpret_cast<const float*>(ml)) : *ml;
          w[k] = SHARED ? load_shared4(po) : *reinterpret_cast<const float4*>(po);
        }
        ok &= v[k].x == v[k].x;
        mb = fmaxf(mb, v[k].x);
      }
      raise(mb);
#pragma unroll
      for (uint32_t k = 0; k < N; k++) add(v[k].x, v[k].y, w[k]);
    }
  }
  __device__ __forceinline__ bool mean(float4& to) const {
    to = make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
    return ok && m > -INFINITY;
  }
};
__device__ __forceinline__ void put_ctx(float* d, float4 v) {  // the caller's rows: any float's alignment
  *reinterpret_cast<f32x4u*>(d) = f32x4u{v.x, v.y, v.z, v.w};
}

// LDS of k8_rows: queries, the own block's keys and values, its weights and sums, the waves' sums.
uint32_t kv8_rows_lds(uint32_t hdp, uint32_t rows) {
  return ((16 + 2 * kKv8Block + rows + 4 * rows) * kv8_pad(hdp) + 16 * 16) * 4;
}

// Workgroup i of a step: its entry and part, the entries' parts laid end to end (so that no workgroup
// is launched for a part that a shorter sequence does not have). Each lane counts one entry's.
// Returns false past the last.
__device__ __forceinline__ bool step_part(const Kv8Args& a, const Kv8Inline& inl, uint32_t i, uint32_t& x, uint32_t& z,
                                          AttnEntry& e) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t e0 = 0; e0 < a.n; e0 += 64) {
    AttnEntry mine{};
    uint32_t n = 0;
    if (e0 + lane < a.n) {
      mine = a.ent ? a.ent[e0 + lane] : inl.e[e0 + lane];
      n = kv8_parts_of(mine.pos, mine.start);
    }
    uint32_t sum = n;  // inclusive prefix
#pragma unroll
    for (uint32_t o = 1; o < 64; o *= 2) {
      const uint32_t v = (uint32_t)__shfl_up((int)sum, o, 64);
      if (lane >= o) sum += v;
    }
    const uint64_t past = __ballot(sum > i);
    if (past) {
      const int l = __builtin_ctzll(past);
      x = e0 + l;
      z = i - (uint32_t)__builtin_amdgcn_readlane((int)(sum - n), l);
      const uint64_t pages = (uint64_t)mine.pages;
      e.pages = (uint32_t*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(pages >> 32), l) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)pages, l));
      e.pos = (uint32_t)__builtin_amdgcn_readlane((int)mine.pos, l);
      e.start = (uint32_t)__builtin_amdgcn_readlane((int)mine.start, l);
      e.page = (uint32_t)__builtin_amdgcn_readlane((int)mine.page, l);
      e.fresh = (uint32_t)__builtin_amdgcn_readlane((int)mine.fresh, l);
      return true;
    }
    i -= (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}

__device__ __forceinline__ float* ctx_row(const Kv8Args& a, const Kv8Run& run, uint32_t h, uint32_t r) {
  const uint32_t G = a.n_heads / a.p.n_kv;
  return a.ctx + ((size_t)(run.i0 + r / G) * a.n_heads + h * G + r % G) * a.p.hd;
}
// Column c of a row whose weights are uniform (four columns; rare).
template <bool STEP, bool SHARED>
__device__ __forceinline__ float4 uniform_row(const Kv8Args& a, const Kv8Run& run, uint32_t h, uint32_t r, uint32_t c) {
  const Kv8Pool& p = a.p;
  const uint32_t hd = p.hd, pos = run.pos0 + r / (a.n_heads / p.n_kv);
  const float* vo = STEP ? kv8_open(p, run.table, h) + (size_t)p.n_kv * kKv8Block * hd
                         : a.own + (((size_t)run.job * 2 + 1) * p.n_kv + h) * kKv8Block * hd;
  float u[4];
  for (uint32_t k = 0; k < 4; k++) u[k] = uniform_mean(p, run.table, h, kv8_start(a, pos), pos, 4 * c + k, vo, hd, STEP && SHARED);
  return make_float4(u[0], u[1], u[2], u[3]);
}

// 256 threads: contexts of a.jrows rows, joined from their parts: kKv8Join parts at a time,
// in order, by hd / 4 threads, then what these give. In a call without this launch (kv8_fused) there
// are no more than the first of those.
template <bool STEP>
__global__ void __launch_bounds__(256) k8_join(Kv8Args a, Kv8Inline inl) {
  __shared__ float4 go[256];
  __shared__ float gm[256], gl[256];
  __shared__ uint32_t bad[256];
  const Kv8Pool& p = a.p;
  const Kv8Part part = rows_parts(a, STEP);
  const uint32_t t = threadIdx.x, hd = p.hd, q4 = hd / 4, c = t % q4, g = t / q4;
  const uint32_t nr = a.jrows, per = 256 / q4 / nr;  // rows, and threads' groups a row
  const uint32_t w = g / per, i = blockIdx.x * nr + w, r = i % part.R, h = i / part.R % p.n_kv, x = i / part.R / p.n_kv;
  Kv8Run run{};
  if (w < nr && x < part.nx) {
    if (STEP) {
      const AttnEntry e = a.ent ? a.ent[x] : inl.e[x];
      run = Kv8Run{x, 1, e.pos, 0, (uint32_t)((e.pages - p.tables) / p.ppseq)};
    } else {
      run = a.run[x];
    }
  }
  const bool in = r < run.n * (a.n_heads / p.n_kv);
  const uint32_t n = in ? kv8_parts_of(run.pos0, kv8_start(a, run.pos0)) : 0;
  bad[t] = 0;
  __syncthreads();
  Joined all;
  for (uint32_t s0 = 0; s0 < a.nparts; s0 += per * kKv8Join) {
    Joined j;
    const uint32_t s = s0 + g % per * kKv8Join;
    j.parts<false, 8>(part, s, min(n, s + kKv8Join), part.row(0, x, h, r), hd, c);
    if (!j.ok) bad[w] = 1;
    go[t] = j.o;
    gm[t] = j.m;
    gl[t] = j.l;
    __syncthreads();
    if (in && g % per == 0)
      for (uint32_t k = t; k < t + per * q4; k += q4) {
        all.raise(gm[k]);
        all.add(gm[k], gl[k], go[k]);
      }
    __syncthreads();
  }
  if (!in || g % per) return;
  float4 o;
  if (!all.mean(o) || bad[w]) o = uniform_row<STEP, false>(a, run, h, r, c);
  put_ctx(ctx_row(a, run, h, r) + 4 * c, o);
}

// STEP: groups are entries, and the token is appended here. ONE: one workgroup takes both
// the own block and what is before it (at most kKv8Split positions), and writes the context.
// grid: (groups * n_kv, 1, parts), in a step without ONE (parts of all entries * n_kv). The kv
// head runs fastest: a page's heads follow each other, and workgroups of one head alone would
// read an eighth of the memory's channels at a time (8 sequences at 65000: 228 us that way).
template <int NS, bool STEP, bool ONE>
__global__ void __launch_bounds__(256, NS <= 6 ? 2 : 1) k8_rows(Kv8Args a, Kv8Inline inl) {
  constexpr uint32_t HDP = 32 * NS, NP = NS / 2, QS = kv8_pad(HDP), Q4 = HDP / 4;
  extern __shared__ float4 lds_v4[];
  __shared__ uint32_t red[8];
  __shared__ float own_m[16], own_l[16], wm[4][16], wl[4][16];
  const Kv8Pool& p = a.p;
  const uint32_t h = blockIdx.x % p.n_kv, t = threadIdx.x, hd = p.hd, G = a.n_heads / p.n_kv;
  const uint32_t lane = t & 63, n16 = lane & 15, kg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  uint32_t x = blockIdx.x / p.n_kv, z = blockIdx.z;
  Kv8Run run;
  AttnEntry e{};
  if (STEP) {
    if (ONE) e = a.ent ? a.ent[x] : inl.e[x];
    else if (!step_part(a, inl, x, x, z, e)) return;
    run = Kv8Run{x, 1, e.pos, 0, (uint32_t)((e.pages - p.tables) / p.ppseq)};
  } else {
    run = a.run[x];
  }
  constexpr uint32_t hs = QS;
  const uint32_t rows = run.n * G;
  float* qs = reinterpret_cast<float*>(lds_v4);  // [16][QS]
  float* kt = qs + 16 * QS;                      // [16][hs], then the values
  float* vt = kt + kKv8Block * hs;
  float* ps = vt + kKv8Block * hs;               // [16][16]
  float* oo = ps + 16 * 16;                      // [rows][hs]
  float* wo = oo + rows * hs;                    // [4][rows][QS]
  auto start_of = [&](uint32_t pos) { return kv8_start(a, pos); };
  const uint32_t own = run.pos0 / kKv8Block * kKv8Block, last = run.pos0 + run.n - 1;
  const uint32_t base = start_of(run.pos0) / kKv8Block * kKv8Block;
  const uint32_t lo = base + (ONE || z == 0 ? 0 : z - 1) * kKv8Split, hi = min(own, lo + kKv8Split);
  const Kv8Part part = rows_parts(a, STEP);
  auto prow = [&](uint32_t r) { return part.row(z, x, h, r); };
  if (!ONE && z && lo >= hi) return;  // a call's group without that part
  const bool mine = ONE || z == 0;
  auto done = [&] {  // the last of the group's workgroups joins its parts; otherwise k8_join does
    if (!a.fused) return;
    if (last_part(a.done + (size_t)x * p.n_kv + h, kv8_parts_of(run.pos0, start_of(run.pos0)), &red[0]))
      for (uint32_t i = t; i < rows * Q4; i += 256) {
        const uint32_t r = i / Q4, c = i % Q4;
        if (4 * c >= hd) continue;
        Joined j;
        j.parts<true, 8>(part, 0, kv8_parts_of(run.pos0, start_of(run.pos0)), part.row(0, x, h, r), hd, c);
        float4 o;
        if (!j.mean(o)) o = uniform_row<STEP, true>(a, run, h, r, c);
        put_ctx(ctx_row(a, run, h, r) + 4 * c, o);
      }
  };
  auto put4 = [&](float* d, float4 v) {
    if (a.fused) store_shared4(d, v);
    else *reinterpret_cast<float4*>(d) = v;
  };
  auto put2 = [&](float2* d, float2 v) {
    if (a.fused) store_shared2(reinterpret_cast<float*>(d), v);
    else *d = v;
  };
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
  // queries, turned (a call's were in the launch before)
  constexpr int QN = (16 * Q4 + 255) / 256;
  float4 qv[QN];
  auto q_at = [&](int y, uint32_t& r, uint32_t& c) {
    const uint32_t i = t + 256 * y;
    r = i / Q4;
    c = i % Q4;
    return r < rows;
  };
#pragma unroll
  for (int y = 0; y < QN; y++) {
    uint32_t r, c;
    qv[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!q_at(y, r, c) || 4 * c >= hd) continue;
    const uint32_t i = run.i0 + r / G, g = h * G + r % G;
    if (STEP) qv[y] = four_of(a.q + (size_t)i * a.q_stride + g * hd + 4 * c, a.nsl, a.sl_stride);
    else qv[y] = *reinterpret_cast<const float4*>(a.qr + ((size_t)i * a.n_heads + g) * hd + 4 * c);
  }
  BlockRows<NS> ob;
  const uint32_t block = run.pos0 / kKv8Block, r0 = run.pos0 % kKv8Block;
  if (mine) {
    if (STEP) {
      if (e.fresh && h == 0 && t == 0) e.pages[run.pos0 / p.bs] = e.page;  // for the calls after this one
      ob.load(a, run.table, r0, 1, h, [&](uint32_t) { return x; });
    } else {
      const float* src = a.own + ((size_t)run.job * 2 * p.n_kv + h) * kKv8Block * hd;
#pragma unroll
      for (uint32_t y = 0; y < NS; y++) {
        const uint32_t i = t + 256 * y;
        ob.v[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (4 * ob.col(i) < hd)
          ob.v[y] = *reinterpret_cast<const float4*>(src + (size_t)ob.value(i) * p.n_kv * kKv8Block * hd + ob.row(i) * hd + 4 * ob.col(i));
      }
    }
  }
#pragma unroll
  for (int y = 0; y < QN; y++) {
    uint32_t r, c;
    if (!q_at(y, r, c)) continue;
    if (STEP && 4 * c < hd) qv[y] = turned(p, qv[y], c, run.pos0);
    *reinterpret_cast<float4*>(qs + r * QS + 4 * c) = qv[y];
  }
  if (mine) {
    if (STEP) {
      ob.turn_keys(p, block, r0, 1);
      ob.template put_global<!ONE>(p, p.open + (size_t)run.table * 2 * p.n_kv * kKv8Block * hd, h, r0 + 1);
    }
    ob.put(kt, vt, hs);
    if (STEP && r0 == kKv8Block - 1) {
      const uint2 m = ob.largest(red);  // with a barrier
      hold_block<NS>(p, kv8_block(p, e.page, block, h), kt, vt, hs, m);
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
    for (uint32_t y = t; y < rows * Q4; y += 256) {
      const uint32_t r = y / Q4, d = 4 * (y % Q4), pr = run.pos0 + r / G, st = start_of(pr);
      if (d >= hd) continue;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t j = st > own ? st - own : 0; j <= pr - own; j++) {
        const float w = ps[r * 16 + j];
        const float4 v = *reinterpret_cast<const float4*>(vt + j * hs + d);
        o = make_float4(fmaf(w, v.x, o.x), fmaf(w, v.y, o.y), fmaf(w, v.z, o.z), fmaf(w, v.w, o.w));
      }
      if (ONE) *reinterpret_cast<float4*>(oo + r * hs + d) = o;
      else put4(part.o + prow(r) * hd + d, o);
    }
    if (!ONE) {
      if (t < rows) put2(part.ml + prow(t), make_float2(own_m[t], own_l[t]));
      done();
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
      const float ck = sk * cq;
      float svn = sv;
      const uint32_t k0 = kb + kKv8Block * kg;
      const bool edge = kb < start_max || kb + 64 > hi;  // the same in every lane
      kb += 256;
      const bool more = kb < hi;
      if (more) {
        find(kb);
        load_k();
      }
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const uint32_t pk = k0 + 4 * q + r;
            if (pk < start_n || pk >= hi) s[q][r] = -INFINITY;
          }
        if (k0 >= hi || k0 + kKv8Block <= start_n) {  // no position of the block is attended to
          svn = 0.0f;
        }
      }
      // scores are s ck (a block's scale is a lane's, and not negative: the largest s is the largest score),
      // weights 2^(s ck - M), at most 2^14: M is the largest score less 14. A NaN or +inf score
      // makes L a NaN.
      float mt = -INFINITY;
#pragma unroll
      for (int q = 0; q < 4; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) mt = fmaxf(mt, s[q][r]);
      const bool none = mt == -INFINITY;  // as 0 times it is a NaN
      mt = fmaxf(M, max16_32(none ? mt : mt * ck) - 14.0f);
      const int en = max(ev, (int)max16_32((float)pow2_of(svn)));
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
            const float sv1 = s[2 * y + q][r];
            float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(sv1, ck, -mu));
            if (edge && sv1 == -INFINITY) pv = 0.0f;
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
  bad |= L != L || M == INFINITY;
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
  for (uint32_t y = t; y < rows * Q4; y += 256) {
    const uint32_t r = y / Q4, d = 4 * (y % Q4);
    if (d >= hd) continue;
    float m = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float4& to, const float4& w, float f) {
      to = make_float4(to.x + w.x * f, to.y + w.y * f, to.z + w.z * f, to.w + w.w * f);
    };
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
        add(v, *reinterpret_cast<const float4*>(wo + (w * rows + r) * QS + d), f);
      }
    if (bd) m = __uint_as_float(kBadRow);
    if (!ONE) {
      put4(part.o + prow(r) * hd + d, v);
      if (d == 0) put2(part.ml + prow(r), make_float2(m, l));
      continue;
    }
    // the own block's part and this one, as Joined adds them
    const float m0 = own_m[r], mm = fmaxf(m0, m);
    const uint32_t pr = run.pos0 + r / G;
    float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (bd || m0 != m0 || mm == -INFINITY) {
      float u[4];
      for (uint32_t k = 0; k < 4; k++) u[k] = uniform_mean(p, run.table, h, start_of(pr), pr, d + k, vt, hs);
      c = make_float4(u[0], u[1], u[2], u[3]);
    } else {
      float ls = 0.0f;
      if (m0 > -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(m0 - mm);
        ls += own_l[r] * f;
        add(c, *reinterpret_cast<const float4*>(oo + r * hs + d), f);
      }
      if (m > -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(m - mm);
        ls += l * f;
        add(c, v, f);
      }
      c = make_float4(c.x / ls, c.y / ls, c.z / ls, c.w / ls);
    }
    put_ctx(ctx_row(a, run, h, r) + d, c);
  }
  if (!ONE) done();
}

// One row again, by the first 256 threads of the workgroup (all of which call it), in f32: 64
// positions at a time, four threads a score. ls: 64 floats, po: 256 float4 of LDS. Threads
// t < hd / 4 return the row's columns 4 t .. 4 t + 3.
__device__ __forceinline__ float4 row_again(const Kv8Args& a, const Kv8Run& run, uint32_t h, uint32_t r, float* ls, float4* po) {
  const Kv8Pool& p = a.p;
  const uint32_t t = threadIdx.x, lane = t & 63, hd = p.hd, G = a.n_heads / p.n_kv, pos = run.pos0 + r / G;
  const uint32_t start = kv8_start(a, pos), own = pos / kKv8Block * kKv8Block;
  const float* q = a.qr + ((size_t)(run.i0 + r / G) * a.n_heads + h * G + r % G) * hd;
  const uint32_t job = run.job + pos / kKv8Block - run.pos0 / kKv8Block;
  const float* ko = a.own + ((size_t)job * 2 * p.n_kv + h) * kKv8Block * hd;
  const float* vo = ko + (size_t)p.n_kv * kKv8Block * hd;
  const uint32_t q4 = hd / 4, ng = 256 / q4, g = t / q4, c = t % q4;
  float M = -INFINITY, L = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  bool uniform = false;
  for (uint32_t c0 = start / kKv8Block * kKv8Block; c0 <= pos && !uniform; c0 += 64) {
    const uint32_t pk = c0 + t / 4;
    float s = 0.0f;
    const bool in = pk >= start && pk <= pos;
    if (in && t < 256) {
      const size_t u = pk < own ? kv8_block(p, kv8_page(p, run.table, pk / kKv8Block), pk / kKv8Block, h) : 0;
      for (uint32_t d = t % 4; d < hd; d += 4)
        s = fmaf(q[d], pk < own ? (float)((int)kv8_codes(p, u)[kv8_key(p.hdp, pk % kKv8Block, d)] - 128) : ko[(pk - own) * hd + d], s);
      if (pk < own) s *= p.scales[2 * u];
    }
    s += __shfl_xor(s, 1, 64);
    s += __shfl_xor(s, 2, 64);
    __syncthreads();
    if (t < 256 && t % 4 == 0) ls[t / 4] = in ? s * (a.scale * kLog2e) : -INFINITY;
    __syncthreads();
    const float v = ls[lane];
    if (__ballot(v != v || v == INFINITY)) uniform = true;  // every wave sees the same scores
    const float mc = wave64_max(v);
    if (uniform || mc == -INFINITY) continue;
    const float mn = fmaxf(M, mc), f = __builtin_amdgcn_exp2f(M - mn), pv = __builtin_amdgcn_exp2f(v - mn);
    M = mn;
    L = L * f + wave64_sum(pv);
    __syncthreads();
    if (t < 64) ls[t] = pv;
    __syncthreads();
    o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    if (g < ng)
      for (uint32_t j = g; j < 64; j += ng) {
        const uint32_t pj = c0 + j;
        if (pj < start || pj > pos) continue;
        const float w = ls[j];
        float4 b;
        if (pj < own) {
          const size_t u = kv8_block(p, kv8_page(p, run.table, pj / kKv8Block), pj / kKv8Block, h);
          const uint8_t* cv = kv8_codes(p, u) + kKv8Block * p.hdp + pj % kKv8Block;
          const float sv = p.scales[2 * u + 1];
          auto at = [&](uint32_t d) { return (float)((int)cv[d * kKv8Block] - 128) * sv; };
          b = make_float4(at(4 * c), at(4 * c + 1), at(4 * c + 2), at(4 * c + 3));
        } else {
          b = *reinterpret_cast<const float4*>(vo + (pj - own) * hd + 4 * c);
        }
        o = make_float4(fmaf(w, b.x, o.x), fmaf(w, b.y, o.y), fmaf(w, b.z, o.z), fmaf(w, b.w, o.w));
      }
  }
  if (uniform || M == -INFINITY) {
    if (t >= q4) return o;
    float u[4];
    for (uint32_t k = 0; k < 4; k++) u[k] = uniform_mean(p, run.table, h, start, pos, 4 * t + k, vo, hd);
    return make_float4(u[0], u[1], u[2], u[3]);
  }
  __syncthreads();
  if (t < 256) po[t] = o;
  __syncthreads();
  if (t < q4) {
    for (uint32_t k = 1; k < ng; k++) {
      const float4 b = po[k * q4 + t];
      o = make_float4(o.x + b.x, o.y + b.y, o.z + b.z, o.w + b.w);
    }
    o = make_float4(o.x / L, o.y / L, o.z / L, o.w / L);
  }
  return o;
}

// The rows r0 + i of the bits i that are set in marks [8].
__device__ __forceinline__ void rows_again(const Kv8Args& a, const Kv8Run& run, uint32_t h, uint32_t r0, const uint32_t* marks, float* ls,
                           float4* po) {
  for (uint32_t k = 0; k < 8; k++)
    for (uint32_t left = marks[k]; left; left &= left - 1) {
      const uint32_t r = r0 + 32 * k + __builtin_ctz(left), t = threadIdx.x;
      const float4 v = row_again(a, run, h, r, ls, po);
      if (t < a.p.hd / 4) put_ctx(ctx_row(a, run, h, r) + 4 * t, v);
      __syncthreads();
    }
}

// ---------------------------------------------------------------------------------
// Attention of a prompt: tiles of up to 256 (token, query head) rows of one kv head, of heads wider
// than 128 up to 128.
//
// One workgroup a (kv head, tile, split of the keys), 8 waves (4) of 32 rows. The groups above
// read a kv head's codes once for 16 rows; here 64 positions (32) at a time go through LDS for
// all rows, converted to fp16 once (16 KB of keys and 16 of values transposed, two buffers: the
// next step's codes are in registers while this one's products run). Products as above, on
// v_mfma_f32_32x32x16_f16: S^T = K Q^T with the rows of A in such an order that a lane's
// 16 scores of 32 positions are 8 consecutive ones of each of two blocks, its own half of
// the second product's B operand; O^T = V^T P^T.
//
// Split 0 takes the rows' own blocks after its positions, or by itself, 32 positions at a time: f32
// rows, scaled by a power of two for each block, as two fp16 each, three of the four products of
// two such sums (the fourth is 2^-22 of the first). A row that meets a score that is NaN or +inf, or whose own block
// has a value that is not finite, is marked and summed again by itself in f32 (row_again).
//
// The sums of 32 rows of 256 are half the registers that a SIMD has for one wave: it runs alone, its
// accumulation registers hold them and the queries' first halves, and nothing but the order of its
// instructions hides the reads of LDS (1024 tokens at 8192, 8 heads of 256 on one: 309 us as the
// compiler puts them, 254 so; in groups 559).
//
// Grid x is the kv head: workgroups go round-robin over the 8 XCDs, so with 8 kv heads a
// head's codes are read into one XCD's L2.
// ---------------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float max32(float v) {
  const LanePair p = xor32_pair(v);
  return fmaxf(p.a, p.b);
}
__device__ __forceinline__ Kv8Part tile_parts(const Kv8Args& a) {
  return parts_of(a, a.tpart, a.tsplits, a.ntile, kv8_tile_rows(a.p.hd));
}

template <int NS>
__global__ void __launch_bounds__(NS <= 4 ? 512 : 256, NS <= 4 ? 2 : 1) k8_tile(Kv8Args a) {
  constexpr uint32_t W = kv8_tile_rows(32 * NS) / 32, NT = 64 * W;             // waves and threads
  constexpr uint32_t HDP = 32 * NS, KS = HDP / 16, NP = NS / 2, CH = HDP / 8;  // CH: 16-byte columns of a key row
  constexpr uint32_t KX = CH % 16 == 0 ? 16 : CH % 8 == 0 ? 8 : 4;             // keys' column x is at x ^ (key % KX)
  constexpr uint32_t PS = NS <= 4 ? 64 : 32, NB = PS / 16;                     // a step's positions, and blocks
  constexpr uint32_t KB = PS * HDP * 2, VB = PS * 2, BUF = 2 * KB;             // bytes of its keys; of a dim's values; of a buffer
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BUF];
  __shared__ u32x4 qlo[W * KS * 64];  // the queries' second halves: in registers they would spill
  __shared__ float2 sc[2][NB];
  __shared__ uint32_t marks[8];  // rows to be summed again, a bit each
  const Kv8Pool& p = a.p;
  const uint32_t h = blockIdx.x, x = blockIdx.y, z = blockIdx.z, t = threadIdx.x, hd = p.hd, G = a.n_heads / p.n_kv;
  // the own blocks by split 0, or by one of their own before the others
  const bool owns = z == 0;
  const uint32_t zk = z - a.town;
  const uint32_t lane = t & 63, l32 = lane & 31, hf = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  auto uni = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane(v); };
  const Kv8Run* T = a.run + a.nrun + x;
  const uint32_t i0 = uni(T->i0), ntok = uni(T->n), pos0 = uni(T->pos0), table = uni(T->table), job0 = uni(T->job);
  const uint32_t rows = ntok * G, last = pos0 + ntok - 1;
  auto start_of = [&](uint32_t pos) { return kv8_start(a, pos); };
  auto own_of = [](uint32_t pos) { return pos / kKv8Block * kKv8Block; };
  const uint32_t base = own_of(start_of(pos0)), lo = base + zk * a.tkeys, hi = a.town && owns ? 0 : min(own_of(last), lo + a.tkeys);
  const uint32_t row = 32 * wave + l32, rr = min(row, rows - 1), pos = pos0 + rr / G;
  const uint32_t start = start_of(pos), own = own_of(pos);
  const Kv8Part part = tile_parts(a);
  const size_t prow = part.row(z, x, h, row);
  const bool mine = row < rows, busy = 32 * wave < rows;
  if (!owns && lo >= hi) return;
  // what the wave's rows attend to of the held blocks: from its first row's start to its last row's own block
  const uint32_t pw0 = pos0 + min(32 * wave, rows - 1) / G, pw1 = pos0 + min(32 * wave + 31, rows - 1) / G;
  const uint32_t w_lo = start_of(pw0), w_hi = min(own_of(pw1), hi), w_in0 = start_of(pw1), w_in1 = min(own_of(pw0), hi);

  // the thread's 16 byte pieces of codes of a tile: of block sb, column sx of its HDP; the pages
  // looked up a tile ahead
  constexpr uint32_t NY = (NB * HDP + NT - 1) / NT;
  auto vcol = [](uint32_t d, uint32_t x) { return (x ^ (PS == 64 ? d % 8 : d / 2 % 4)) * 16; };
  auto sb = [&](uint32_t y) { return (t + NT * y) / HDP; };
  auto sx = [&](uint32_t y) { return (t + NT * y) % HDP; };
  auto staged = [&](uint32_t y) { return NB * HDP % NT == 0 || sb(y) < NB; };
  size_t unit[NY];
  auto find = [&](uint32_t kb) {
#pragma unroll
    for (uint32_t y = 0; y < NY; y++) {
      const uint32_t b = min(kb + kKv8Block * min(sb(y), NB - 1), hi - 1) / kKv8Block;
      unit[y] = kv8_block(p, kv8_page(p, table, b), b, h);
    }
  };
  uint4 kc[NY], vc[NY];
  float2 sv2[NY];
  auto load = [&]() {
#pragma unroll
    for (uint32_t y = 0; y < NY; y++) {
      const uint8_t* c = p.codes + unit[y] * (2 * kKv8Block * HDP) + sx(y) * 16;
      if (staged(y)) {
        kc[y] = *reinterpret_cast<const uint4*>(c);
        vc[y] = *reinterpret_cast<const uint4*>(c + kKv8Block * HDP);
        sv2[y] = reinterpret_cast<const float2*>(p.scales)[unit[y]];
      }
    }
  };
  uint32_t krow[NY], kcol[NY];  // the keys' row in its block and first 16-byte column
#pragma unroll
  for (uint32_t y = 0; y < NY; y++) {
    const uint32_t c = sx(y);
    if (NS % 2 && c >= 64 * NP) {
      krow[y] = (c - 64 * NP) / 2;
      kcol[y] = 8 * NP + 2 * (c % 2);
    } else {
      krow[y] = c % 64 / 4;
      kcol[y] = 8 * (c / 64) + 2 * (c % 4);
    }
  }
  auto store = [&](uint32_t b) {
    uint8_t* buf = lds + b * BUF;
#pragma unroll
    for (uint32_t y = 0; y < NY; y++) {
      if (!staged(y)) continue;
      const uint32_t s4 = sb(y), c = sx(y), key = kKv8Block * s4 + krow[y];
      uint8_t *kd = buf + key * HDP * 2, *vd = buf + KB + c * VB;
      *reinterpret_cast<f16x8*>(kd + ((kcol[y] ^ (key % KX)) * 16)) = codes8(kc[y].x, kc[y].y);
      *reinterpret_cast<f16x8*>(kd + (((kcol[y] + 1) ^ (key % KX)) * 16)) = codes8(kc[y].z, kc[y].w);
      *reinterpret_cast<f16x8*>(vd + vcol(c, 2 * s4)) = codes8(vc[y].x, vc[y].y);
      *reinterpret_cast<f16x8*>(vd + vcol(c, 2 * s4 + 1)) = codes8(vc[y].z, vc[y].w);
      if (c == 0) sc[b][s4] = sv2[y];
    }
  };
  const bool any = !(a.town && owns) && lo < hi;
  if (any) {
    find(lo);
    load();
    find(lo + PS);
  }
  // queries: the wave's B operand
  f16x8 qh[KS];
  u32x4* qlw = qlo + wave * KS * 64 + lane;
  auto ql = [&](uint32_t st) { return __builtin_bit_cast(f16x8, qlw[64 * st]); };
  float cq;
  bool odd;
  {
    const float* q = a.qr + ((size_t)(i0 + rr / G) * a.n_heads + h * G + rr % G) * hd;
    float4 v[KS][2];
    float m = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t s = 0; s < KS; s++)
#pragma unroll
      for (uint32_t y = 0; y < 2; y++) {
        const uint32_t d = 16 * s + 8 * hf + 4 * y;
        v[s][y] = d < hd ? *reinterpret_cast<const float4*>(q + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (float f : {v[s][y].x, v[s][y].y, v[s][y].z, v[s][y].w}) {
          m = fmaxf(m, fabsf(f));
          top = max(top, __float_as_uint(f) & 0x7fffffffu);
        }
      }
    m = max32(m);
    odd = max32(top >= 0x7f800000u ? 1.0f : 0.0f) != 0.0f;
    const int eq = odd ? 0 : pow2_of(m);
    const float up = pow2(9 - eq);
    cq = a.scale * kLog2e * pow2(max(eq - 9, -126));
#pragma unroll
    for (uint32_t s = 0; s < KS; s++) {
      float f[8] = {v[s][0].x * up, v[s][0].y * up, v[s][0].z * up, v[s][0].w * up,
                    v[s][1].x * up, v[s][1].y * up, v[s][1].z * up, v[s][1].w * up};
      if (odd)
        for (int y = 0; y < 8; y++) f[y] = 0.0f;
      f16x8 lo8;
      split8(f, qh[s], lo8);
      qlw[64 * s] = __builtin_bit_cast(u32x4, lo8);  // a lane's own
      if (NS > 4) {  // in accumulation registers, which the products read as well
        u32x4 b = __builtin_bit_cast(u32x4, qh[s]);
        asm("" : "+a"(b));
        qh[s] = __builtin_bit_cast(f16x8, b);
      }
    }
  }
  f32x16 o[NS];
#pragma unroll
  for (int d = 0; d < NS; d++) o[d] = (f32x16)(0.0f);
  float M = -INFINITY, L = 0.0f;
  int ev = -100;
  // a lane's key of the MFMA's row l32: 8 consecutive ones of a block to a half
  const uint32_t arow = 16 * (l32 / 16) + 8 * (l32 / 4 % 2) + 4 * (l32 / 8 % 2) + l32 % 4;
  // Products s, each eight of a block whose scores are s ck and whose values have the scale svn, to
  // weights and the row's sums. Weights are 2^(score - M): M is 8 below the largest score when
  // it is set, and set again only where a score is more than 13 above it, as the sums' values'
  // unit 2^ev is only where a scale is 4 times it or more. So few tiles rescale the sums (with
  // M the running maximum, a tile of a long span in two did), weights times scales stay
  // below 2^15, and what is left of them after the first fp16 has 11 bits down to 2^-11 of the
  // largest weight, then to 2^-33 of it. A NaN or +inf score makes L a NaN. Masked products are
  // -inf (every ck is above 0).
  auto soften = [&](const float* s, const int n, const float* ck, const float* svn, int en, float* w) {
    float mt = -INFINITY;
#pragma unroll
    for (int y = 0; y < n / 8; y++) {
      float mb = s[8 * y];
#pragma unroll
      for (int r = 1; r < 8; r++) mb = fmaxf(mb, s[8 * y + r]);
      mt = fmaxf(mt, mb * ck[y]);
    }
    mt = max32(mt);
    const bool up = mt - M > 13.0f;
    if (__ballot(up) || en > ev + 1) {
      asm volatile("");
      const float mn = up ? mt - 8.0f : M, was = M;
      M = mn;
      float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(was - mn);
      L *= f;
      if (en > ev + 1) {
        f *= pow2(max(ev - en, -126));
        ev = en;
      }
#pragma unroll
      for (int d = 0; d < NS; d++) {
        if (NS > 4) asm volatile("" : "+a"(o[d]));
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] *= f;
        if (NS > 4) asm volatile("" : "+a"(o[d]));
      }
    }
    const float mu = M == -INFINITY ? 0.0f : M, un = pow2(-ev);
    float sum = 0.0f;
#pragma unroll
    for (int y = 0; y < n / 8; y++) {
      const float vn = svn[y] * un;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        const float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * y + r], ck[y], -mu));
        sum += pv;
        w[8 * y + r] = pv * vn;
      }
    }
    L += sum;
  };
  // PS held positions from kb on, in a buffer
  auto step = [&](uint32_t kb, uint32_t b) {
    const uint8_t* kbuf = lds + b * BUF;
    float s[PS / 2], w[PS / 2], svn[NB], ck[NB];
    int en = -100;
#pragma unroll
    for (uint32_t y = 0; y < NB; y++) {
      const uint32_t c = (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_int(sc[b][y].x));
      const uint32_t v = (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_int(sc[b][y].y));
      ck[y] = above0(__uint_as_float(c) * cq);
      svn[y] = __uint_as_float(v);
      en = max(en, pow2_of(__uint_as_float(v)));
    }
    f32x16 acc[PS / 32];
#pragma unroll
    for (uint32_t y = 0; y < PS / 32; y++) acc[y] = (f32x16)(0.0f);
#pragma unroll
    for (uint32_t st = 0; st < KS; st++) {
      const f16x8 lo8 = ql(st);
#pragma unroll
      for (uint32_t y = 0; y < PS / 32; y++) {
        const uint32_t key = 32 * y + arow;
        const f16x8 kf = *reinterpret_cast<const f16x8*>(kbuf + key * HDP * 2 + (((2 * st + hf) ^ (key % KX)) * 16));
        acc[y] = mfma32(kf, lo8, acc[y]);
        acc[y] = mfma32(kf, qh[st], acc[y]);
      }
    }
    if (NS > 4) {  // reads of LDS three products' operands ahead
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (uint32_t st = 0; st < KS; st++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
    }
#pragma unroll
    for (uint32_t y = 0; y < PS / 32; y++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) s[16 * y + r] = acc[y][r];
    if (kb < w_in0 || kb + PS > w_in1) {  // some row of the wave does not attend to all
      asm volatile("");                   // a branch: the selects of every tile were a fifth of its instructions
      const uint32_t top = min(own, hi);
#pragma unroll
      for (uint32_t y = 0; y < NB; y++) {
        const uint32_t k0 = kb + 16 * y;
        if (k0 >= top || k0 + 16 <= start) {
          svn[y] = 0.0f;
          ck[y] = 1.0f;
        }
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
          const uint32_t pk = k0 + 8 * hf + r;
          if (pk < start || pk >= top) s[8 * y + r] = -INFINITY;
        }
      }
    }
    soften(s, PS / 2, ck, svn, en, w);
#pragma unroll
    for (uint32_t y = 0; y < NB; y++) {
      f16x8 wh, wl;
      split8(w + 8 * y, wh, wl);
#pragma unroll
      for (uint32_t d = 0; d < NS; d++) {
        const uint32_t dr = 32 * d + l32;
        const f16x8 vf = *reinterpret_cast<const f16x8*>(kbuf + KB + dr * VB + vcol(dr, 2 * y + hf));
        o[d] = mfma32(vf, wl, o[d]);
        o[d] = mfma32(vf, wh, o[d]);
      }
    }
    if (NS > 4) {
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
      for (uint32_t st = 0; st < NB * NS; st++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 2, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      }
    }
  };
  if (any) store(0);
  __syncthreads();
  uint32_t buf = 0;
  for (uint32_t kb = lo; any && kb < hi; kb += PS, buf ^= 1) {
    const bool more = kb + PS < hi;
    if (NS > 4)  // the sums in accumulation registers here and in soften: 256 moves a step otherwise
#pragma unroll
      for (int d = 0; d < NS; d++) asm("" : "+a"(o[d]));
    if (more) {
      load();
      if (kb + 2 * PS < hi) find(kb + 2 * PS);
    }
    if (busy && kb < w_hi && kb + PS > w_lo) {
      step(kb, buf);
    }
    if (more) store(buf ^ 1);
    __syncthreads();
  }
  if (owns) {
    // the rows' own blocks, two at a time: planes of keys [2][32][HDP], of values transposed [2][HDP][32]
    constexpr uint32_t PK = 32 * HDP * 2, PV = HDP * 32 * 2;
    const uint32_t b_end = last / kKv8Block;
    for (uint32_t b0 = pos0 / kKv8Block; b0 <= b_end; b0 += 2) {
      float2 up[2];  // powers of two: keys and values below 2^10
      float svn[2], skn[2];
      bool wild[2];
#pragma unroll
      for (uint32_t y = 0; y < 2; y++) {
        const uint32_t job = job0 + min(b0 + y, b_end) - pos0 / kKv8Block;
        const float2 m = a.own_max[(size_t)job * p.n_kv + h];
        wild[y] = !(fabsf(m.x) < INFINITY) || !(fabsf(m.y) < INFINITY);
        const int ek = wild[y] ? 0 : pow2_of(m.x), em = wild[y] ? 0 : pow2_of(m.y);
        up[y] = make_float2(pow2(9 - ek), pow2(9 - em));
        skn[y] = pow2(max(ek - 9, -126));
        svn[y] = pow2(max(em - 9, -126));
      }
      auto src = [&](uint32_t y, uint32_t kv) {  // rows of block b0 + y
        const uint32_t job = job0 + min(b0 + y, b_end) - pos0 / kKv8Block;
        return a.own + (((size_t)job * 2 + kv) * p.n_kv + h) * kKv8Block * hd;
      };
      __syncthreads();
      for (uint32_t it = t; it < 32 * (HDP / 4); it += NT) {
        const uint32_t key = it / (HDP / 4), d = it % (HDP / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (d < hd && !(key < 16 ? wild[0] : wild[1])) v = *reinterpret_cast<const float4*>(src(key / 16, 0) + key % 16 * hd + d);
        const float u = key < 16 ? up[0].x : up[1].x;
        const float f[4] = {v.x * u, v.y * u, v.z * u, v.w * u};
        uint8_t* dst = lds + key * HDP * 2 + (((d / 8) ^ (key % KX)) * 16 + 8 * (d / 4 % 2));
        uint32_t hi2[2], lo2[2];
#pragma unroll
        for (int y = 0; y < 2; y++) split2(f[2 * y], f[2 * y + 1], hi2[y], lo2[y]);
        *reinterpret_cast<u32x2*>(dst) = u32x2{hi2[0], hi2[1]};
        *reinterpret_cast<u32x2*>(dst + PK) = u32x2{lo2[0], lo2[1]};
      }
      for (uint32_t it = t; it < 16 * (HDP / 4); it += NT) {
        const uint32_t kp = it % 16, d = it / 16 * 4, key = 2 * kp;
        float4 v0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v1 = v0;
        if (d < hd && !(key < 16 ? wild[0] : wild[1])) {  // 0 times a NaN would reach the other block's rows
          const float* s = src(key / 16, 1) + key % 16 * hd + d;
          v0 = *reinterpret_cast<const float4*>(s);
          v1 = *reinterpret_cast<const float4*>(s + hd);
        }
        const float u = key < 16 ? up[0].y : up[1].y;
        const float f[4][2] = {{v0.x * u, v1.x * u}, {v0.y * u, v1.y * u}, {v0.z * u, v1.z * u}, {v0.w * u, v1.w * u}};
#pragma unroll
        for (uint32_t y = 0; y < 4; y++) {
          uint32_t hi2, lo2;
          split2(f[y][0], f[y][1], hi2, lo2);
          uint8_t* dst = lds + 2 * PK + (d + y) * 64 + (((key / 8) ^ ((d + y) / 2 % 4)) * 16 + 2 * (key % 8));
          *reinterpret_cast<uint32_t*>(dst) = hi2;
          *reinterpret_cast<uint32_t*>(dst + PV) = lo2;
        }
      }
      __syncthreads();
      const uint32_t k0 = b0 * kKv8Block;
      if (busy && k0 <= pw1 && k0 + 32 > own_of(pw0)) {
        f32x16 acc = (f32x16)(0.0f);
#pragma unroll
        for (uint32_t st = 0; st < KS; st++) {
          const uint8_t* at = lds + arow * HDP * 2 + (((2 * st + hf) ^ (arow % KX)) * 16);
          const f16x8 kh = *reinterpret_cast<const f16x8*>(at), kl = *reinterpret_cast<const f16x8*>(at + PK);
          acc = mfma32(kl, qh[st], acc);
          acc = mfma32(kh, ql(st), acc);
          acc = mfma32(kh, qh[st], acc);
        }
        float s[16], w[16], sn[2], ck[2];
#pragma unroll
        for (uint32_t y = 0; y < 2; y++) {
          const bool at = own == k0 + 16 * y;
          odd |= at && wild[y];
          sn[y] = at && !wild[y] ? svn[y] : 0.0f;
          ck[y] = above0(skn[y] * cq);
#pragma unroll
          for (uint32_t r = 0; r < 8; r++) {
            const uint32_t pk = k0 + 16 * y + 8 * hf + r;
            s[8 * y + r] = at && !wild[y] && pk <= pos && pk >= start ? acc[8 * y + r] : -INFINITY;
          }
        }
        soften(s, 16, ck, sn, max(pow2_of(svn[0]), pow2_of(svn[1])), w);
#pragma unroll
        for (uint32_t y = 0; y < 2; y++) {
          f16x8 wh, wl;
          split8(w + 8 * y, wh, wl);
#pragma unroll
          for (uint32_t d = 0; d < NS; d++) {
            const uint32_t dr = 32 * d + l32;
            const uint8_t* at = lds + 2 * PK + dr * 64 + (((2 * y + hf) ^ (dr / 2 % 4)) * 16);
            const f16x8 vh = *reinterpret_cast<const f16x8*>(at), vl = *reinterpret_cast<const f16x8*>(at + PV);
            o[d] = mfma32(vl, wh, o[d]);
            o[d] = mfma32(vh, wl, o[d]);
            o[d] = mfma32(vh, wh, o[d]);
          }
        }
      }
    }
  }
  {
    const LanePair l = xor32_pair(L);
    L = l.a + l.b;
  }
  odd = max32(odd ? 1.0f : 0.0f) != 0.0f || L != L || M == INFINITY;
  const float fo = pow2(ev);
  auto four = [&](uint32_t d, uint32_t j, float f) {  // columns 32 d + 8 j + 4 hf on
    return make_float4(o[d][4 * j] * f, o[d][4 * j + 1] * f, o[d][4 * j + 2] * f, o[d][4 * j + 3] * f);
  };
  if (a.tsplits > 1) {
    if (!mine) return;
    if (hf == 0) part.ml[prow] = make_float2(odd ? __uint_as_float(kBadRow) : M, L);
#pragma unroll
    for (uint32_t d = 0; d < NS; d++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t c = 32 * d + 8 * j + 4 * hf;
        if (c < hd) *reinterpret_cast<float4*>(part.o + prow * hd + c) = four(d, j, fo);
      }
    return;
  }
  // the only split: the context itself
  if (t < 8) marks[t] = 0;
  __syncthreads();
  const Kv8Run run{i0, ntok, pos0, job0, table};
  if (mine) {
    const bool again = odd || M == -INFINITY;
    if (again && hf == 0) atomicOr(&marks[row / 32], 1u << (row % 32));
#pragma unroll
    for (uint32_t d = 0; d < NS; d++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t c = 32 * d + 8 * j + 4 * hf;
        const float4 v = four(d, j, fo);
        if (c < hd && !again) put_ctx(ctx_row(a, run, h, row) + c, make_float4(v.x / L, v.y / L, v.z / L, v.w / L));
      }
  }
  __syncthreads();
  rows_again(a, run, h, 0, marks, reinterpret_cast<float*>(lds + 4096), reinterpret_cast<float4*>(lds));
}

// grid (tiles * n_kv, 256 / rows a workgroup), 256 threads: the splits of a tile's rows joined,
// a thread per four columns of a row.
__global__ void __launch_bounds__(256) k8_join_tile(Kv8Args a) {
  __shared__ float4 po[256];
  __shared__ float ls[64];
  __shared__ uint32_t marks[8];
  const Kv8Pool& p = a.p;
  const uint32_t x = blockIdx.x / p.n_kv, h = blockIdx.x % p.n_kv, t = threadIdx.x, hd = p.hd, q4 = hd / 4, rpw = 256 / q4;
  const uint32_t G = a.n_heads / p.n_kv;
  const Kv8Run run = a.run[a.nrun + x];
  const Kv8Part part = tile_parts(a);
  const uint32_t r0 = blockIdx.y * rpw, r = r0 + t / q4, c = t % q4, rows = run.n * G;
  if (r0 >= rows) return;
  if (t < 8) marks[t] = 0;
  __syncthreads();
  if (t / q4 < rpw && r < rows) {
    const uint32_t last = run.pos0 + run.n - 1, first = kv8_start(a, run.pos0);
    const uint32_t held = (last / kKv8Block * kKv8Block - first / kKv8Block * kKv8Block + a.tkeys - 1) / a.tkeys;
    const uint32_t n = max(1u, a.town + held);
    Joined j;
    j.parts<false, 2>(part, 0, n, part.row(0, x, h, r), hd, c);
    float4 v;
    if (j.mean(v)) put_ctx(ctx_row(a, run, h, r) + 4 * c, v);
    else if (c == 0) atomicOr(&marks[(r - r0) / 32], 1u << ((r - r0) % 32));
  }
  __syncthreads();
  rows_again(a, run, h, r0, marks, ls, po);
}

// grid (chunks * n_kv), 256 threads: rows of one block, from its codes or from the open rows.
template <int NS>
__global__ void __launch_bounds__(256) k8_read(Kv8Pool p, const Kv8Rows* rows, Kv8RowsInline inl, float* k, float* v) {
  constexpr uint32_t HDP = 32 * NS, Q4 = HDP / 4;
  __shared__ uint32_t vt[kKv8Block * HDP / 4];
  const uint32_t h = blockIdx.x % p.n_kv, i0 = blockIdx.x / p.n_kv, t = threadIdx.x, hd = p.hd, kvd = p.n_kv * hd;
  const Kv8Rows r = rows ? rows[i0] : inl.r[i0];
  auto put = [&](float* to, uint32_t row, uint32_t c, float4 w) {  // the caller's rows: any float's alignment
    *reinterpret_cast<f32x4u*>(to + (size_t)(r.i0 + row) * kvd + h * hd + 4 * c) = f32x4u{w.x, w.y, w.z, w.w};
  };
  if (!r.whole) {
    const float* src = kv8_open(p, r.table, h);
#pragma unroll
    for (uint32_t y = 0; y < NS; y++) {
      const uint32_t i = t + 256 * y, val = i / (16 * Q4), row = i / Q4 % 16, c = i % Q4;
      if (row < r.n && 4 * c < hd)
        put(val ? v : k, row, c, *reinterpret_cast<const float4*>(src + (size_t)val * p.n_kv * kKv8Block * hd + (r.r0 + row) * hd + 4 * c));
    }
    return;
  }
  const size_t u = kv8_block(p, kv8_page(p, r.table, r.block), r.block, h);
  const uint8_t* codes = kv8_codes(p, u);
  const float2 sc = reinterpret_cast<const float2*>(p.scales)[u];
  auto value = [](uint32_t w, uint32_t b, float s) { return (float)((int)(w >> 8 * b & 255u) - 128) * s; };
  const uint32_t* vw = reinterpret_cast<const uint32_t*>(codes + kKv8Block * HDP);
  constexpr uint32_t W = kKv8Block * HDP / 4;
#pragma unroll
  for (uint32_t y = 0; y < W; y += 256) {
    const uint32_t i = t + y, row = i / Q4, c = i % Q4;
    if (W % 256 && i >= W) break;
    vt[i] = vw[i];  // word d * 4 + row / 4
    if (row < r.n && 4 * c < hd) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + kv8_key(HDP, r.r0 + row, 4 * c));
      put(k, row, c, make_float4(value(w, 0, sc.x), value(w, 1, sc.x), value(w, 2, sc.x), value(w, 3, sc.x)));
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t y = 0; y < W; y += 256) {
    const uint32_t i = t + y, row = i / Q4, c = i % Q4;
    if (W % 256 && i >= W) break;
    if (row < r.n && 4 * c < hd) {
      const uint32_t a = r.r0 + row;
      float f[4];
#pragma unroll
      for (uint32_t d = 0; d < 4; d++) f[d] = value(vt[(4 * c + d) * 4 + a / 4], a % 4, sc.y);
      put(v, row, c, make_float4(f[0], f[1], f[2], f[3]));
    }
  }
}

// grid (blocks * n_kv), 256 threads: rows r0 .. r0 + n - 1 of a held block become open rows.
__global__ void __launch_bounds__(256) k8_reopen(Kv8Pool p, Kv8RowsInline inl) {
  const Kv8Rows r = inl.r[blockIdx.x / p.n_kv];
  const uint32_t h = blockIdx.x % p.n_kv, hd = p.hd;
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

template <int NS, bool STEP>
void launch_rows(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) {
  // what 16 rows of the widest heads of this build take, set once; a call asks for its own rows'
  static const bool set = [] {
    const int most = (int)kv8_rows_lds(32 * NS, 16);
    return hipFuncSetAttribute((const void*)k8_rows<NS, STEP, true>, hipFuncAttributeMaxDynamicSharedMemorySize, most) == hipSuccess &&
           hipFuncSetAttribute((const void*)k8_rows<NS, STEP, false>, hipFuncAttributeMaxDynamicSharedMemorySize, most) == hipSuccess;
  }();
  (void)set;
  const bool one = a.nparts == 2;  // one workgroup a group and kv head
  const uint32_t G = a.n_heads / a.p.n_kv, rows = STEP ? G : kv8_group_tokens(G) * G, nx = STEP ? a.n : a.nrun;
  const uint32_t lds = kv8_rows_lds(a.p.hdp, rows);
  const dim3 grid(a.p.n_kv * (STEP && !one ? a.items : nx), 1, STEP || one ? 1 : a.nparts);
  auto kernel = one ? k8_rows<NS, STEP, true> : k8_rows<NS, STEP, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, a, inl);
  if (one || a.fused) return;
  const uint32_t n = a.p.n_kv * nx * rows;
  Kv8Args j = a;
  j.jrows = kv8_join_rows(a.p.hd, a.nparts, n);
  hipLaunchKernelGGL(k8_join<STEP>, dim3((n + j.jrows - 1) / j.jrows), dim3(256), 0, st, j, inl);
}

// f of the build for the heads' width
template <class F>
void by_width(uint32_t hdp, F&& f) {
  switch (hdp / 32) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 6: f(std::integral_constant<int, 6>()); break;
    default: f(std::integral_constant<int, 8>()); break;
  }
}

template <bool STEP>
hipError_t launch_rows_of(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) {
  by_width(a.p.hdp, [&](auto ns) { launch_rows<ns(), STEP>(a, inl, st); });
  return hipGetLastError();
}

}  // namespace

bool kv8_fits(const Kv8Args& a, bool step) {
  const uint64_t kv = a.p.n_kv, G = a.n_heads / kv;
  // workgroups along x, of 256 threads
  if (step) return kv * a.items <= kMaxWgs && (uint64_t)a.n * a.n_heads <= kMaxWgs;
  return kv * a.njob <= kMaxWgs && a.nrun * kv * kv8_group_tokens(G) * G <= kMaxWgs && kv * a.ntile <= kMaxWgs &&
         a.nparts <= kMaxGridYz && a.ntile <= kMaxGridYz;
}

hipError_t launch_kv8_step(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) { return launch_rows_of<true>(a, inl, st); }

hipError_t launch_kv8_call(const Kv8Args& a, const Kv8CallInline& inl, hipStream_t st) {
  const dim3 jobs(a.njob * a.p.n_kv, 1, a.qr ? 1 + (a.n_heads / a.p.n_kv + 3) / 4 : 1);
  by_width(a.p.hdp, [&](auto ns) {
    if (a.hjob) k8_append<ns(), OfHost><<<jobs, dim3(256), 0, st>>>(a, OfHost{});
    else k8_append<ns(), Kv8CallInline><<<jobs, dim3(256), 0, st>>>(a, inl);
  });
  if (!a.ctx) return hipGetLastError();
  if (a.ntile) {
    const dim3 grid(a.p.n_kv, a.ntile, a.tsplits);
    const uint32_t rpw = 256 / (a.p.hd / 4);
    by_width(a.p.hdp, [&](auto ns) {
      hipLaunchKernelGGL(k8_tile<ns()>, grid, dim3(2 * kv8_tile_rows(32 * ns())), 0, st, a);
    });
    if (a.tsplits > 1)
      hipLaunchKernelGGL(k8_join_tile, dim3(a.ntile * a.p.n_kv, (kv8_tile_rows(a.p.hd) + rpw - 1) / rpw), dim3(256), 0, st, a);
  }
  return a.nrun ? launch_rows_of<false>(a, Kv8Inline{}, st) : hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8Pool& p, const Kv8Rows* rows, const Kv8RowsInline& inl, uint32_t nrows, float* k,
                           float* v, hipStream_t st) {
  by_width(p.hdp, [&](auto ns) {
    hipLaunchKernelGGL(k8_read<ns()>, dim3(nrows * p.n_kv), dim3(256), 0, st, p, rows, inl, k, v);
  });
  return hipGetLastError();
}

hipError_t launch_kv8_reopen(const Kv8Pool& p, const Kv8RowsInline& inl, uint32_t nrows, hipStream_t st) {
  hipLaunchKernelGGL(k8_reopen, dim3(nrows * p.n_kv), dim3(256), 0, st, p, inl);
  return hipGetLastError();
}

}  // namespace gmoe
