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

// The 16 rows kt, vt [16][hd] (in LDS) of one block and head to codes and scales, by 256
// threads; red: 8 words of LDS. Every thread calls it after a barrier that follows the rows'.
__device__ void hold_block(const Kv8Pool& p, size_t unit, const float* kt, const float* vt, uint32_t* red) {
  const uint32_t t = threadIdx.x, n = kKv8Block * p.hd;
  uint32_t mk = 0, mv = 0;  // as bits: NaN above infinity above every number
  for (uint32_t x = t; x < n; x += 256) {
    mk = max(mk, __float_as_uint(kt[x]) & 0x7fffffffu);
    mv = max(mv, __float_as_uint(vt[x]) & 0x7fffffffu);
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
  auto inv = [](uint32_t m) { return m == 0 || m >= 0x7f800000u ? 0.0 : 127.0 / (double)__uint_as_float(m); };
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
    for (uint32_t b = 0; b < 4; b++) w |= (d + b < p.hd ? code(kt[r * p.hd + d + b], ik) : 128u) << 8 * b;
    *reinterpret_cast<uint32_t*>(dst + kv8_key(p.hdp, r, d)) = w;
  }
  uint32_t* vd = reinterpret_cast<uint32_t*>(dst + kKv8Block * p.hdp);
  for (uint32_t x = t; x < kKv8Block * p.hdp / 4; x += 256) {
    const uint32_t d = x / 4, r = x % 4 * 4;
    uint32_t w = 0;
    for (uint32_t b = 0; b < 4; b++) w |= (d < p.hd ? code(vt[(r + b) * p.hd + d], iv) : 128u) << 8 * b;
    vd[x] = w;
  }
  if (t == 0) {
    p.scales[2 * unit] = scale(mk);
    p.scales[2 * unit + 1] = scale(mv);
  }
}

// A job's rows of kv head h: earlier ones from the open rows, the call's from k (rotated) and v.
__device__ void job_rows(const Kv8Args& a, const Kv8Job& j, uint32_t h, float* kt, float* vt) {
  const Kv8Pool& p = a.p;
  const uint32_t t = threadIdx.x, hd = p.hd, half = hd / 2;
  const float* old = kv8_open(p, j.table, h);
  for (uint32_t x = t; x < j.r0 * hd; x += 256) {
    kt[x] = old[x];
    vt[x] = old[(size_t)p.n_kv * kKv8Block * hd + x];
  }
  for (uint32_t x = t; x < j.n * half; x += 256) {
    const uint32_t r = j.r0 + x / half, c = x % half;
    const size_t from = (size_t)j.ent[r] * a.kv_stride + h * hd;
    double cs, sn;
    turn(p.turns[c], j.block * kKv8Block + r, cs, sn);
    const float2 k = pair_of(a.k + from, c, a.nsl, a.sl_stride), v = pair_of(a.v + from, c, a.nsl, a.sl_stride);
    reinterpret_cast<float2*>(kt)[r * half + c] = rotated(k.x, k.y, cs, sn);
    reinterpret_cast<float2*>(vt)[r * half + c] = v;
  }
  for (uint32_t x = t + (j.r0 + j.n) * hd; x < kKv8Block * hd; x += 256) kt[x] = vt[x] = 0.0f;
}
__device__ void put_open(const Kv8Pool& p, const Kv8Job& j, uint32_t h, const float* kt, const float* vt) {
  float* to = kv8_open(p, j.table, h);
  for (uint32_t x = threadIdx.x; x < (j.r0 + j.n) * p.hd; x += 256) {
    to[x] = kt[x];
    to[(size_t)p.n_kv * kKv8Block * p.hd + x] = vt[x];
  }
}

// grid (njob, n_kv), 256 threads: a block of the call's positions, one kv head. The job of a
// sequence's first block writes the open rows of its last one, after it has read those that
// were there.
__global__ void __launch_bounds__(256) k8_append(Kv8Args a) {
  extern __shared__ float lds_f[];
  __shared__ uint32_t red[8];
  const Kv8Pool& p = a.p;
  const uint32_t h = blockIdx.y, t = threadIdx.x, n = kKv8Block * p.hd;
  float *kt = lds_f, *vt = kt + n;
  const Kv8Job j = a.hjob[blockIdx.x];
  if (h == 0 && a.run)
    for (uint32_t x = blockIdx.x * 256 + t; x < a.nrun; x += gridDim.x * 256) a.run[x] = a.hrun[x];
  if (h == 0 && t == 0 && (j.flags & kKv8Fresh))
    p.tables[(size_t)j.table * p.ppseq + j.block / (p.bs / kKv8Block)] = j.page;
  job_rows(a, j, h, kt, vt);
  __syncthreads();
  if (a.own) {
    float* own = a.own + ((size_t)blockIdx.x * 2 * p.n_kv + h) * n;
    for (uint32_t x = t; x < n; x += 256) {
      own[x] = kt[x];
      own[(size_t)p.n_kv * n + x] = vt[x];
    }
  }
  if (j.flags & kKv8Whole) hold_block(p, kv8_block(p, j.page, j.block, h), kt, vt, red);
  if (!(j.flags & kKv8First)) return;
  if (j.last != blockIdx.x) {
    __syncthreads();
    const Kv8Job l = a.hjob[j.last];
    job_rows(a, l, h, kt, vt);
    __syncthreads();
    put_open(p, l, h, kt, vt);
  } else {
    put_open(p, j, h, kt, vt);
  }
}

// grid (n, n_kv), 256 threads: one token's query heads of one kv head over its whole span,
// 64 positions at a time. STEP: the token is also appended here; otherwise its block's rows
// are those of its job (a.own).
template <bool STEP>
__global__ void __launch_bounds__(256) k8_attend(Kv8Args a, Kv8Inline inl) {
  extern __shared__ float lds_f[];
  __shared__ uint32_t red[8];
  __shared__ float ps[kAttnMaxGroup][64], ml[kAttnMaxGroup][3];
  __shared__ uint32_t bad;
  const Kv8Pool& p = a.p;
  const uint32_t i = blockIdx.x, h = blockIdx.y, t = threadIdx.x, hd = p.hd, half = hd / 2, G = a.n_heads / p.n_kv;
  float *kt = lds_f, *vt = kt + kKv8Block * hd, *qs = vt + kKv8Block * hd;
  uint32_t pos, table, start;
  if (STEP) {
    const AttnEntry e = a.ent ? a.ent[i] : inl.e[i];
    pos = e.pos;
    start = e.start;
    table = (uint32_t)((e.pages - p.tables) / p.ppseq);
    Kv8Job j{};
    j.table = table;
    j.block = pos / kKv8Block;
    j.page = e.page;
    j.r0 = pos % kKv8Block;
    j.n = 1;
    for (uint32_t r = 0; r < kKv8Block; r++) j.ent[r] = i;
    if (e.fresh && h == 0 && t == 0) e.pages[pos / p.bs] = e.page;
    job_rows(a, j, h, kt, vt);
    __syncthreads();
    if (j.r0 == kKv8Block - 1) hold_block(p, kv8_block(p, j.page, j.block, h), kt, vt, red);
    put_open(p, j, h, kt, vt);
  } else {
    uint32_t r = 0;
    while (i - a.run[r].i0 >= a.run[r].n) r++;
    const Kv8Run run = a.run[r];
    pos = run.pos0 + i - run.i0;
    start = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
    table = run.table;
    const uint32_t job = run.job + pos / kKv8Block - run.pos0 / kKv8Block, n = kKv8Block * hd;
    const float* own = a.own + ((size_t)job * 2 * p.n_kv + h) * n;
    for (uint32_t x = t; x < n; x += 256) {
      kt[x] = own[x];
      vt[x] = own[(size_t)p.n_kv * n + x];
    }
  }
  for (uint32_t x = t; x < G * half; x += 256) {
    double cs, sn;
    turn(p.turns[x % half], pos, cs, sn);
    const float2 q = pair_of(a.q + (size_t)i * a.q_stride + (h * G + x / half) * hd, x % half, a.nsl, a.sl_stride);
    reinterpret_cast<float2*>(qs)[x] = rotated(q.x, q.y, cs, sn);
  }
  if (t == 0) bad = 0;
  if (t < G) {
    ml[t][0] = -INFINITY;
    ml[t][1] = 0.0f;
  }
  float o[16];  // items (g, d) = t, t + 256, ... of the group's [G][hd]
  for (int x = 0; x < 16; x++) o[x] = 0.0f;
  __syncthreads();
  const uint32_t own0 = pos / kKv8Block * kKv8Block;
  for (int pass = 0; pass < 2; pass++) {  // the second: uniform weights
    for (uint32_t c0 = start / kKv8Block * kKv8Block; c0 <= pos; c0 += 64) {
      const uint32_t j = t / 4, pj = c0 + j;
      const bool in = pj >= start && pj <= pos;
      const uint8_t* codes = nullptr;
      float sk = 1.0f;
      if (in && pj < own0) {
        const size_t u = kv8_block(p, kv8_page(p, table, pj / kKv8Block), pj / kKv8Block, h);
        codes = kv8_codes(p, u);
        sk = p.scales[2 * u];
      }
      for (uint32_t g = 0; g < G; g++) {
        float s = 0.0f;
        if (in)
          for (uint32_t d = t % 4; d < hd; d += 4)
            s = fmaf(qs[g * hd + d], codes ? (float)((int)codes[kv8_key(p.hdp, pj % kKv8Block, d)] - 128) : kt[pj % kKv8Block * hd + d], s);
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        if (t % 4 == 0) ps[g][j] = pass ? (in ? 0.0f : -INFINITY) : in ? s * sk * a.scale : -INFINITY;
      }
      __syncthreads();
      for (uint32_t g = t >> 6; g < G; g += 4) {
        const uint32_t lane = t & 63;
        const float s = ps[g][lane], mo = ml[g][0];
        if (__ballot(s != s || s == INFINITY) && lane == 0) atomicOr(&bad, 1u << g);
        const float m = fmaxf(mo, wave64_max(s));
        const float e = m > -INFINITY && s > -INFINITY ? gm_expf(s - m) : 0.0f;
        ps[g][lane] = e;
        const float l = wave64_sum(e);
        if (lane == 0) {
          const float f = mo > -INFINITY ? gm_expf(mo - m) : 0.0f;
          ml[g][0] = m;
          ml[g][1] = fmaf(ml[g][1], f, l);
          ml[g][2] = f;
        }
      }
      __syncthreads();
      for (uint32_t x = 0; x * 256 + t < G * hd; x++) {
        const uint32_t g = (x * 256 + t) / hd, d = (x * 256 + t) % hd;
        float acc = o[x] * ml[g][2];
        for (uint32_t b = 0; b < 4 && c0 + 16 * b <= pos; b++) {
          const uint32_t blk = c0 / kKv8Block + b;
          if (blk * kKv8Block == own0) {
            for (uint32_t r = 0; r <= pos % kKv8Block; r++)
              if (ps[g][16 * b + r] != 0.0f) acc = fmaf(ps[g][16 * b + r], vt[r * hd + d], acc);
          } else {
            const size_t u = kv8_block(p, kv8_page(p, table, blk), blk, h);
            const uint8_t* vc = kv8_codes(p, u) + kKv8Block * p.hdp + d * kKv8Block;
            float s = 0.0f;
            bool any = false;
            for (uint32_t r = 0; r < kKv8Block; r++) {
              s = fmaf(ps[g][16 * b + r], (float)((int)vc[r] - 128), s);
              any |= blk * kKv8Block + r >= start;
            }
            if (any) acc = fmaf(s, p.scales[2 * u + 1], acc);
          }
        }
        o[x] = acc;
      }
      __syncthreads();
    }
    // a row without a score above -inf, or with one that is NaN or +inf: again, every score 0
    for (uint32_t g = 0; g < G; g++)
      if (t == 0 && ml[g][0] == -INFINITY) bad |= 1u << g;
    __syncthreads();
    const uint32_t b = bad;
    for (uint32_t x = 0; x * 256 + t < G * hd; x++) {
      const uint32_t g = (x * 256 + t) / hd;
      if ((pass != 0) == ((b >> g & 1) != 0)) a.ctx[((size_t)i * a.n_heads + h * G) * hd + x * 256 + t] = o[x] / ml[g][1];
      o[x] = 0.0f;
    }
    if (!b) return;
    __syncthreads();
    if (t < G) {
      ml[t][0] = -INFINITY;
      ml[t][1] = 0.0f;
    }
    __syncthreads();
  }
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

uint32_t rows_lds(const Kv8Args& a) { return (2 * kKv8Block + a.n_heads / a.p.n_kv) * a.p.hd * 4; }

}  // namespace

hipError_t launch_kv8_step(const Kv8Args& a, const Kv8Inline& inl, hipStream_t st) {
  hipLaunchKernelGGL(k8_attend<true>, dim3(a.n, a.p.n_kv), dim3(256), rows_lds(a), st, a, inl);
  return hipGetLastError();
}

hipError_t launch_kv8_call(const Kv8Args& a, hipStream_t st) {
  hipLaunchKernelGGL(k8_append, dim3(a.njob, a.p.n_kv), dim3(256), 2 * kKv8Block * a.p.hd * 4, st, a);
  if (a.ctx) hipLaunchKernelGGL(k8_attend<false>, dim3(a.n, a.p.n_kv), dim3(256), rows_lds(a), st, a, Kv8Inline{});
  return hipGetLastError();
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
