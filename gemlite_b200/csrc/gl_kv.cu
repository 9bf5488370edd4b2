// Quantised key/value cache: write (head norms, rotary positions and quantisation in one pass) and read back, sm_100a.
//
// Both kernels move bytes: every operand is read once, every output written once.  A row (one token's head) is spread over
// head_dim / 8 lanes of 8 channels each, so that norms and maxima are three or four shuffles.  The write takes a lane's channels as
// two pieces of 4 (8-byte loads), which puts both channels of a rotated pair into one lane; the read takes them as one piece of codes
// (8 bytes, 4 in the 4-bit format) and stores 16 bytes or more of the output.
#include "gl_kv_attend.cuh"

int gl_kv_check(const char* fn, const gl_kv_args* a) {
  if (a == nullptr) GL_FAIL(GL_E_INVALID, "%s: null argument struct", fn);
  if (a->format < GL_KV_FP8 || a->format > GL_KV_INT4) GL_FAIL(GL_E_INVALID, "%s: unknown cache format %d", fn, a->format);
  if (a->head_dim != 64 && a->head_dim != 128) GL_FAIL(GL_E_UNSUPPORTED, "%s: head_dim %d (64 and 128 are supported)", fn, a->head_dim);
  if (a->num_pages <= 0 || a->page_size <= 0 || a->n_kv_heads <= 0 || a->batch < 0 || a->max_pages < 0 || a->n_tokens < 0 || a->max_len < 0 || a->max_new < 0)
    GL_FAIL(GL_E_INVALID, "%s: bad size (pages %d x %d, kv heads %d, batch %d, table columns %d, tokens %d)", fn, a->num_pages, a->page_size,
            a->n_kv_heads, a->batch, a->max_pages, a->n_tokens);
  // slots are 32-bit numbers: 2^32 rows of keys and values, 74 bytes at least, are more than the GPU's memory
  if ((uint64_t)a->num_pages * (uint64_t)a->n_kv_heads > 0xfffffffeull / (uint64_t)a->page_size)
    GL_FAIL(GL_E_UNSUPPORTED, "%s: %d pages of %d heads x %d tokens (at most 2^32 - 2 rows)", fn, a->num_pages, a->n_kv_heads, a->page_size);
  if (!a->k_codes || !a->v_codes || !a->k_scales || !a->v_scales) GL_FAIL(GL_E_INVALID, "%s: null cache pointer", fn);
  if (((uintptr_t)a->k_codes | (uintptr_t)a->v_codes) & 15) GL_FAIL(GL_E_INVALID, "%s: codes must be 16-byte aligned", fn);
  if (((uintptr_t)a->k_scales | (uintptr_t)a->v_scales | (uintptr_t)a->page_table | (uintptr_t)a->lens | (uintptr_t)a->q_offsets) & 3)
    GL_FAIL(GL_E_INVALID, "%s: scales, page table, lengths and offsets must be 4-byte aligned", fn);
  if (a->format == GL_KV_INT4 && (!a->k_zeros || !a->v_zeros)) GL_FAIL(GL_E_INVALID, "%s: the 4-bit cache needs zeros", fn);
  if (a->batch > 0 && (!a->lens || (a->max_pages > 0 && !a->page_table))) GL_FAIL(GL_E_INVALID, "%s: null page table or lengths", fn);
  if (a->batch > 0 && a->q_offsets == nullptr && a->n_tokens % a->batch != 0)
    GL_FAIL(GL_E_INVALID, "%s: %d tokens do not divide evenly over %d sequences; pass q_offsets", fn, a->n_tokens, a->batch);
  return GL_OK;
}

namespace {

template <typename T> struct Half2Of;
template <> struct Half2Of<__nv_bfloat16> {
  static __device__ __forceinline__ float2 up(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Half2Of<__half> {
  static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

struct WriteParams {
  KvBatch kb;
  const void *q, *k, *v;
  void* q_out;
  const void *q_norm, *k_norm;
  const float* cos_sin;
  const int32_t* positions;
  uint8_t *codes[2], *zeros[2];
  float* scales[2];
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh;
  int32_t hq, rot, table_rows, norm_dtype;
  float eps;
};

// One block per token (and slice of its heads): the token's rotation, its norm weights and its slot are fetched once and
// serve all of its heads.  LPR lanes per row of 8 channels each, taken as two pieces of 4 so that a channel and its partner in the
// rotation are in the same lane.  Queries go four rows at a time: their sums of squares are reduced together, each lane then
// takes the square root and the reciprocal of one row.
//
// The order of the fp32 operations is the one of the formulas, without fused multiply-adds, and the sum of squares is kept in
// fp64: a code next to a rounding border then does not depend on how the row was spread over lanes.
//
// 8192 tokens of 64 + 2 x 8 heads of 128 into fp8 (323 MB): 110 us, 2.9 TB/s (155 us with partners fetched by shuffles and one row
// at a time).  Bound by issue slots (fp64 sums, correctly rounded divisions and roots) and by the latency of a token's loads;
// 80 registers (140 bytes of spills), three blocks per SM.  One token: 4.1 us, four dependent loads.  Fewer than 64 heads of 128 (128 of
// 64) leave lane groups without a row that still go through the arithmetic: 3108 tokens of 24 + 2 x 4 heads of 64 into 4 bits (24 MB) take
// 39 us under ncu.
template <typename T, int LPR> struct Rows {
  static constexpr int D = LPR * 8;
  struct Raw { uint2 p, q; };
  int a, b;                                    // first channel of each piece
  __device__ __forceinline__ Raw load(const T* row) const { return Raw{*reinterpret_cast<const uint2*>(row + a), *reinterpret_cast<const uint2*>(row + b)}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&x)[8]) {
    const uint32_t w[4] = {r.p.x, r.p.y, r.q.x, r.q.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = Half2Of<T>::up(w[j]);
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
  }
};

// a lane's 8 weights: two pieces of 4
__device__ __forceinline__ void load_weights(const void* w, int dtype, int a, int b, float (&v)[8]) {
  if (dtype == GL_FP32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = reinterpret_cast<const float*>(w)[a + j];
      v[4 + j] = reinterpret_cast<const float*>(w)[b + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = reinterpret_cast<const uint16_t*>(w)[a + j], y = reinterpret_cast<const uint16_t*>(w)[b + j];
      v[j] = dtype == GL_BF16 ? __uint_as_float(x << 16) : __half2float(__ushort_as_half((unsigned short)x));
      v[4 + j] = dtype == GL_BF16 ? __uint_as_float(y << 16) : __half2float(__ushort_as_half((unsigned short)y));
    }
  }
}

// x / sqrt(mean x^2 + eps) * w of R rows (1 or 4) of a group of LPR lanes
template <int R, int LPR>
__device__ __forceinline__ void normalise(float (&x)[R][8], const float (&w)[8], float eps, unsigned gmask) {
  const int lane = threadIdx.x % LPR;
  double ss[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ss[r] = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss[r] += (double)x[r][j] * (double)x[r][j];
  }
  double mine = ss[0];
  int o = LPR / 2;
  if constexpr (R == 4) {                      // halves of the group keep two rows each, quarters one
    const bool up = lane & (LPR / 2), up2 = lane & (LPR / 4);
    const double k0 = (up ? ss[2] : ss[0]) + __shfl_xor_sync(gmask, up ? ss[0] : ss[2], LPR / 2);
    const double k1 = (up ? ss[3] : ss[1]) + __shfl_xor_sync(gmask, up ? ss[1] : ss[3], LPR / 2);
    mine = (up2 ? k1 : k0) + __shfl_xor_sync(gmask, up2 ? k0 : k1, LPR / 4);
    o = LPR / 8;
  }
  for (; o > 0; o >>= 1) mine += __shfl_xor_sync(gmask, mine, o);
  const float mean = (float)(mine * (1.0 / (LPR * 8)));
  float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, eps)));
  // bf16 numbers beyond 2^64: their mean square, at most 2^256, goes through fp32 with 2^-128 (eps is nothing beside it)
  if (mean == INFINITY) inv = __fmul_rn(__fdiv_rn(1.0f, __fsqrt_rn((float)(mine * (0x1p-128 / (LPR * 8))))), 0x1p-64f);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float f = R == 1 ? inv : __shfl_sync(gmask, inv, ((threadIdx.x & 31) / LPR) * LPR + (r >> 1) * (LPR / 2) + (r & 1) * (LPR / 4));
#pragma unroll
    for (int j = 0; j < 8; ++j) x[r][j] = __fmul_rn(__fmul_rn(x[r][j], f), w[j]);
  }
}
template <bool INTER> __device__ __forceinline__ void rotate(float (&x)[8], const float (&cs)[4], const float (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = INTER ? x[2 * j] : x[j], b = INTER ? x[2 * j + 1] : x[4 + j];
    x[INTER ? 2 * j : j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
    x[INTER ? 2 * j + 1 : 4 + j] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
  }
}

template <typename T, int LPR, int FMT, bool INTER>
__global__ void __launch_bounds__(256, 3) kv_write_kernel(const WriteParams p) {
  constexpr int D = LPR * 8, GROUPS = 256 / LPR, R = 4;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const unsigned gmask = (LPR == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / LPR * LPR);
  gl_launch_dependents();
  gl_grid_dependency_wait();
  // this lane's channels, and their norm weights
  const bool turns = lane * 8 < p.rot;
  Rows<T, LPR> rows;
  rows.a = INTER || !turns ? lane * 8 : lane * 4;
  rows.b = INTER || !turns ? lane * 8 + 4 : p.rot / 2 + lane * 4;
  const int hq = p.q != nullptr ? p.hq : 0;
  float wq[8], wk[8];
  if (p.q_norm != nullptr) load_weights(p.q_norm, p.norm_dtype, rows.a, rows.b, wq);
  if (p.k_norm != nullptr) load_weights(p.k_norm, p.norm_dtype, rows.a, rows.b, wk);

  for (int n = blockIdx.x; n < p.kb.n_tokens; n += gridDim.x) {
    // what does not depend on the sequence first: the first rows, and the position
    const T* q_src = reinterpret_cast<const T*>(p.q) + n * p.q_sn;
    typename Rows<T, LPR>::Raw raw[R], raw_kv;
    const int hkv = p.kb.hkv, kv_first = (int)(gridDim.y - 1 - blockIdx.y) * GROUPS + group;      // (slices take keys and values from the other end)
    auto fetch_q = [&](int h0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int h = h0 + group + r * gridDim.y * GROUPS;
        raw[r].p = raw[r].q = make_uint2(0, 0);
        if (h < hq) raw[r] = rows.load(q_src + h * p.q_sh);
      }
    };
    auto fetch_kv = [&](int r0) {
      if (r0 < 2 * hkv) raw_kv = rows.load(r0 < hkv ? reinterpret_cast<const T*>(p.k) + n * p.k_sn + r0 * p.k_sh : reinterpret_cast<const T*>(p.v) + n * p.v_sn + (r0 - hkv) * p.v_sh);
    };
    fetch_q(blockIdx.y * GROUPS);
    fetch_kv(kv_first);
    const int at = p.rot > 0 ? p.positions[n] : 0;

    // sequence of row n: how many sequences end at or before it
    int b = 0, i = 0;
    if (p.kb.q_offsets != nullptr) {
      for (int base = 0; base < p.kb.batch; base += 32) {
        const int t = base + (threadIdx.x & 31);
        const unsigned done = __ballot_sync(0xffffffffu, t < p.kb.batch && p.kb.q_offsets[t + 1] <= n);
        b += __popc(done);
        if (done != 0xffffffffu) break;                      // ascending
      }
      if (b >= p.kb.batch || n < p.kb.q_offsets[0]) continue;
      i = n - p.kb.q_offsets[b];
    } else {
      const int t = p.kb.n_tokens / p.kb.batch;
      b = n / t;
      i = n - b * t;
    }
    const int64_t slot0 = kv_slot(p.kb, b, 0, (int64_t)max(p.kb.lens[b], 0) + i);

    // this lane's share of the rotation: the cosine and sine of four pairs
    float cs[4], sn[4];
    bool bad_pos = false;
    if (p.rot > 0) {
      bad_pos = (unsigned)at >= (unsigned)p.table_rows;
      if (turns) {
        const float* t = p.cos_sin + (bad_pos ? 0 : (int64_t)at * p.rot) + lane * 4;
        const float4 c4 = *reinterpret_cast<const float4*>(t), s4 = *reinterpret_cast<const float4*>(t + p.rot / 2);
        cs[0] = c4.x; cs[1] = c4.y; cs[2] = c4.z; cs[3] = c4.w;
        sn[0] = s4.x; sn[1] = s4.y; sn[2] = s4.z; sn[3] = s4.w;
      }
    }
    // ---- queries
    if (hq > 0) {
      T* dst = reinterpret_cast<T*>(p.q_out) + (int64_t)n * hq * D;
      for (int h0 = blockIdx.y * GROUPS; h0 < hq; h0 += gridDim.y * GROUPS * R) {
        float x[R][8];
#pragma unroll
        for (int r = 0; r < R; ++r) rows.unpack(raw[r], x[r]);
        if (h0 + gridDim.y * GROUPS * R < hq) fetch_q(h0 + gridDim.y * GROUPS * R);
        if (p.q_norm != nullptr) normalise<R, LPR>(x, wq, p.eps, gmask);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int h = h0 + group + r * gridDim.y * GROUPS;
          if (turns) rotate<INTER>(x[r], cs, sn);
          if (bad_pos)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[r][j] = __int_as_float(0x7fc00000);
          if (h < hq) {
            *reinterpret_cast<uint2*>(dst + h * D + rows.a) = make_uint2(Half2Of<T>::down(x[r][0], x[r][1]), Half2Of<T>::down(x[r][2], x[r][3]));
            *reinterpret_cast<uint2*>(dst + h * D + rows.b) = make_uint2(Half2Of<T>::down(x[r][4], x[r][5]), Half2Of<T>::down(x[r][6], x[r][7]));
          }
        }
      }
    }
    if (slot0 < 0) continue;

    // ---- keys and values
    for (int r0 = kv_first; r0 < 2 * hkv; r0 += gridDim.y * GROUPS) {
      const int which = r0 < hkv ? 0 : 1, h = which ? r0 - hkv : r0;
      float x[1][8];
      rows.unpack(raw_kv, x[0]);
      fetch_kv(r0 + gridDim.y * GROUPS);
      if (which == 0) {
        if (p.k_norm != nullptr) normalise<1, LPR>(x, wk, p.eps, gmask);
        if (turns) rotate<INTER>(x[0], cs, sn);
        if (bad_pos)                               // channels that do not turn as well: no half-valid rows
#pragma unroll
          for (int j = 0; j < 8; ++j) x[0][j] = __int_as_float(0x7fc00000);
      }
      const int64_t slot = slot0 + (int64_t)h * p.kb.page_size;
      // |x| as integers: infinities and NaN are the largest
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[0][j]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(gmask, top, o));
      const bool finite = top < 0x7f800000u;
      if (FMT == GL_KV_INT4) {
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) { lo = fminf(lo, x[0][j]); hi = fmaxf(hi, x[0][j]); }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
          lo = fminf(lo, __shfl_xor_sync(gmask, lo, o));
          hi = fmaxf(hi, __shfl_xor_sync(gmask, hi, o));
        }
        const float span = __fsub_rn(hi, lo);                      // (of bf16 numbers beyond 2^127 it is no fp32 number)
        const float scale = fmaxf(span < INFINITY ? __fdiv_rn(span, 15.f) : __fsub_rn(__fdiv_rn(hi, 15.f), __fdiv_rn(lo, 15.f)), 1e-6f);
        const float zero = fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.f), 15.f);
        uint32_t o = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float c = fminf(fmaxf(rintf(__fdiv_rn(x[0][j], scale)) + zero, 0.f), 15.f);
          o |= (uint32_t)(int)c << (4 * j);
        }
        if (!finite) o = 0u;
        uint8_t* dst = p.codes[which] + slot * (D / 2);
        *reinterpret_cast<uint16_t*>(dst + rows.a / 2) = (uint16_t)o;
        *reinterpret_cast<uint16_t*>(dst + rows.b / 2) = (uint16_t)(o >> 16);
        if (lane == 0) {
          p.scales[which][slot] = finite ? scale : __int_as_float(0x7fc00000);
          p.zeros[which][slot] = finite ? (uint8_t)(int)zero : (uint8_t)0;
        }
      } else {
        const float qmax = FMT == GL_KV_FP8 ? 448.f : 127.f;
        const float scale = fmaxf(__fdiv_rn(__uint_as_float(top), qmax), 1e-6f);
        uint32_t o[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float c = fminf(fmaxf(__fdiv_rn(x[0][j], scale), -qmax), qmax);
          const uint32_t byte = FMT == GL_KV_FP8 ? (uint32_t)__nv_cvt_float_to_fp8(c, __NV_SATFINITE, __NV_E4M3) : (uint32_t)(uint8_t)(int8_t)(int)rintf(c);
          o[j >> 2] |= byte << (8 * (j & 3));
        }
        uint8_t* dst = p.codes[which] + slot * D;
        *reinterpret_cast<uint32_t*>(dst + rows.a) = finite ? o[0] : 0u;
        *reinterpret_cast<uint32_t*>(dst + rows.b) = finite ? o[1] : 0u;
        if (lane == 0) p.scales[which][slot] = finite ? scale : __int_as_float(0x7fc00000);
      }
    }
  }
}

struct ReadParams {
  KvBatch kb;
  const uint8_t *codes[2], *zeros[2];
  const float* scales[2];
  void* out[2];
  int32_t max_len, heads_shift;
};

// One lane per 8 channels, so that a warp's stores are whole lines of the output; a block takes whole tokens (all heads of one
// follow each other there).  Its rows' slots are looked up once, by one thread each, and every lane has the loads of eight rows, keys
// and values, in flight.  Codes become fp16 numbers two at a time, exactly, and are scaled in fp32.
// 95537 tokens of 8 heads of 128, int4 to bf16 (642 MB): 100 us in a captured graph, 6.4 TB/s, the measured copy bandwidth but for 2 %;
// 107 us (6.0 TB/s) called one by one (four rows in flight: 118 us captured; 16 channels per lane, whose stores fill half lines: 139 us).
template <int D, int FMT, typename O>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p) {
  constexpr int RB = FMT == GL_KV_INT4 ? D / 2 : D, LPR = D / 8, GROUPS = 256 / LPR, N = 8, ROWS = GROUPS * N;
  __shared__ int64_t slots[ROWS];              // -1: zeros
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, hkv = p.kb.hkv;
  const int64_t row0 = (int64_t)blockIdx.x * ROWS, end = (int64_t)p.max_len * hkv;
  gl_launch_dependents();
  gl_grid_dependency_wait();
  for (int b = blockIdx.y; b < p.kb.batch; b += gridDim.y) {
    for (int i = threadIdx.x; i < ROWS; i += 256) {
      const int64_t row = row0 + i;
      const uint32_t t = p.heads_shift >= 0 ? (uint32_t)(row >> p.heads_shift) : (uint32_t)((uint64_t)row / (uint32_t)hkv);
      slots[i] = row < end && (int64_t)t < p.kb.lens[b] ? kv_slot(p.kb, b, (int)(row - (int64_t)t * hkv), t) : -1;
    }
    __syncthreads();
    uint2 u[2][N];
    float scale[2][N];
    uint32_t zero[2][N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t slot = slots[i * GROUPS + group];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        u[w][i] = make_uint2(0, 0);
        scale[w][i] = 0.f;
        zero[w][i] = 0;
        if (slot >= 0) {
          if constexpr (FMT == GL_KV_INT4) {
            u[w][i].x = __ldcs(reinterpret_cast<const uint32_t*>(p.codes[w] + slot * RB) + lane);
            zero[w][i] = p.zeros[w][slot];
          } else {
            u[w][i] = __ldcs(reinterpret_cast<const uint2*>(p.codes[w] + slot * RB) + lane);
          }
          scale[w][i] = p.scales[w][slot];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t row = row0 + i * GROUPS + group;
      if (row >= end) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t h[4];
        if constexpr (FMT == GL_KV_INT4) {
          const uint32_t z = (0x6400u + zero[w][i]) * 0x10001u, c = u[w][i].x;
          uint32_t n[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) n[k] = kv_nibbles(c >> (4 * k), z);      // channels (k, k + 4)
          h[0] = __byte_perm(n[0], n[1], 0x5410);
          h[1] = __byte_perm(n[2], n[3], 0x5410);
          h[2] = __byte_perm(n[0], n[1], 0x7632);
          h[3] = __byte_perm(n[2], n[3], 0x7632);
        } else {
          kv_bytes<FMT>(u[w][i].x, h[0], h[1]);
          kv_bytes<FMT>(u[w][i].y, h[2], h[3]);
        }
        float2 f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[k] = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
          f[k].x *= scale[w][i];
          f[k].y *= scale[w][i];
        }
        O* dst = reinterpret_cast<O*>(p.out[w]) + ((int64_t)b * end + row) * D + lane * 8;
        if constexpr (sizeof(O) == 4) {
          __stcs(reinterpret_cast<float4*>(dst), make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
          __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(f[2].x, f[2].y, f[3].x, f[3].y));
        } else {
          __stcs(reinterpret_cast<uint4*>(dst), make_uint4(Half2Of<O>::down(f[0].x, f[0].y), Half2Of<O>::down(f[1].x, f[1].y), Half2Of<O>::down(f[2].x, f[2].y), Half2Of<O>::down(f[3].x, f[3].y)));
        }
      }
    }
    __syncthreads();                           // the slots may be overwritten
  }
}

template <typename T, int LPR, bool INTER>
int launch_write_fmt(const WriteParams& p, int fmt, dim3 grid, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_FP8, INTER>, grid, dim3(256), 0, st, p)); break;
    case GL_KV_INT8: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_INT8, INTER>, grid, dim3(256), 0, st, p)); break;
    default: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_INT4, INTER>, grid, dim3(256), 0, st, p)); break;
  }
  return GL_OK;
}
template <typename T, int LPR>
int launch_write(const WriteParams& p, bool interleaved, int fmt, dim3 grid, cudaStream_t st) {
  return interleaved ? launch_write_fmt<T, LPR, true>(p, fmt, grid, st) : launch_write_fmt<T, LPR, false>(p, fmt, grid, st);
}
template <int D, typename O>
int launch_read(const ReadParams& p, int fmt, dim3 grid, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: GL_CUDA_CHECK(gl_launch_pdl(kv_read_kernel<D, GL_KV_FP8, O>, grid, dim3(256), 0, st, p)); break;
    case GL_KV_INT8: GL_CUDA_CHECK(gl_launch_pdl(kv_read_kernel<D, GL_KV_INT8, O>, grid, dim3(256), 0, st, p)); break;
    default: GL_CUDA_CHECK(gl_launch_pdl(kv_read_kernel<D, GL_KV_INT4, O>, grid, dim3(256), 0, st, p)); break;
  }
  return GL_OK;
}

}  // namespace

extern "C" int gl_kv_write(const gl_kv_args* a, void* stream) {
  if (int rc = gl_kv_check("gl_kv_write", a)) return rc;
  if (a->x_dtype != GL_FP16 && a->x_dtype != GL_BF16) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_write: dtype %d (fp16 / bf16 only)", a->x_dtype);
  if (a->batch == 0 || a->n_tokens == 0) return GL_OK;
  if (!a->k || !a->v) GL_FAIL(GL_E_INVALID, "gl_kv_write: null keys or values");
  if (a->q && (!a->out || a->n_q_heads <= 0)) GL_FAIL(GL_E_INVALID, "gl_kv_write: queries without an output or heads");
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15) GL_FAIL(GL_E_INVALID, "gl_kv_write: operands must be 16-byte aligned");
  if ((a->q_stride_n | a->q_stride_h | a->k_stride_n | a->k_stride_h | a->v_stride_n | a->v_stride_h) & 7)
    GL_FAIL(GL_E_INVALID, "gl_kv_write: strides must be multiples of 8 elements");
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 16 != 0)
    GL_FAIL(GL_E_INVALID, "gl_kv_write: rot_dim %d must be a multiple of 16 up to head_dim", a->rot_dim);
  if (a->rot_dim > 0 && (!a->cos_sin || !a->positions || a->table_rows <= 0)) GL_FAIL(GL_E_INVALID, "gl_kv_write: the rotation needs positions and a cos / sin table");
  if (a->rot_dim > 0 && ((uintptr_t)a->cos_sin & 15)) GL_FAIL(GL_E_INVALID, "gl_kv_write: the cos / sin table must be 16-byte aligned");
  if ((a->q_norm || a->k_norm) && a->norm_dtype != GL_FP32 && a->norm_dtype != GL_FP16 && a->norm_dtype != GL_BF16)
    GL_FAIL(GL_E_INVALID, "gl_kv_write: norm weights of dtype %d", a->norm_dtype);
  if (((a->q_norm || a->k_norm) && (((uintptr_t)a->q_norm | (uintptr_t)a->k_norm) & (gl_dtype_size(a->norm_dtype) - 1))) || (a->rot_dim > 0 && ((uintptr_t)a->positions & 3)))
    GL_FAIL(GL_E_INVALID, "gl_kv_write: misaligned norm weights or positions");
  WriteParams p;
  p.kb = gl_kv_batch(a);
  p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->out;
  p.q_norm = a->q_norm; p.k_norm = a->k_norm; p.cos_sin = a->cos_sin; p.positions = a->positions;
  p.codes[0] = (uint8_t*)a->k_codes; p.codes[1] = (uint8_t*)a->v_codes;
  p.zeros[0] = a->k_zeros; p.zeros[1] = a->v_zeros;
  p.scales[0] = a->k_scales; p.scales[1] = a->v_scales;
  p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h; p.k_sn = a->k_stride_n; p.k_sh = a->k_stride_h; p.v_sn = a->v_stride_n; p.v_sh = a->v_stride_h;
  p.hq = a->n_q_heads; p.rot = a->rot_dim; p.table_rows = a->table_rows; p.norm_dtype = a->norm_dtype;
  p.eps = a->eps;
  // few tokens: their heads are spread over blocks until every SM has a few; many: one block walks a token's heads
  const int lpr = a->head_dim / 8, groups = 256 / lpr;
  const int64_t slices = gl_cdiv(a->q ? a->n_q_heads : 0, groups) + gl_cdiv(2 * a->n_kv_heads, groups), want = gl_cdiv((int64_t)gl_num_sms() * 8, a->n_tokens);
  const int64_t walk = (int64_t)gl_num_sms() * 12;
  const dim3 grid((unsigned)(a->n_tokens < walk ? a->n_tokens : walk), (unsigned)(slices < want ? slices : want));
  cudaStream_t st = (cudaStream_t)stream;
  if (a->x_dtype == GL_BF16)
    return lpr == 16 ? launch_write<__nv_bfloat16, 16>(p, a->interleaved != 0, a->format, grid, st) : launch_write<__nv_bfloat16, 8>(p, a->interleaved != 0, a->format, grid, st);
  return lpr == 16 ? launch_write<__half, 16>(p, a->interleaved != 0, a->format, grid, st) : launch_write<__half, 8>(p, a->interleaved != 0, a->format, grid, st);
}

extern "C" int gl_kv_read(const gl_kv_args* a, void* stream) {
  if (int rc = gl_kv_check("gl_kv_read", a)) return rc;
  if (a->x_dtype != GL_FP16 && a->x_dtype != GL_BF16 && a->x_dtype != GL_FP32) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_read: output dtype %d", a->x_dtype);
  if (a->batch == 0 || a->max_len == 0) return GL_OK;
  if (!a->out || !a->out_v || (((uintptr_t)a->out | (uintptr_t)a->out_v) & 15)) GL_FAIL(GL_E_INVALID, "gl_kv_read: null or misaligned output");
  if ((int64_t)a->max_len * a->n_kv_heads > 0xffffffffll) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_read: %d tokens of %d heads", a->max_len, a->n_kv_heads);
  ReadParams p;
  p.kb = gl_kv_batch(a);
  p.codes[0] = (const uint8_t*)a->k_codes; p.codes[1] = (const uint8_t*)a->v_codes;
  p.zeros[0] = a->k_zeros; p.zeros[1] = a->v_zeros;
  p.scales[0] = a->k_scales; p.scales[1] = a->v_scales;
  p.out[0] = a->out; p.out[1] = a->out_v;
  p.max_len = a->max_len;
  p.heads_shift = (a->n_kv_heads & (a->n_kv_heads - 1)) == 0 ? __builtin_ctz((unsigned)a->n_kv_heads) : -1;
  const int rows = 256 / (a->head_dim / 8) * 8;
  const dim3 grid((unsigned)gl_cdiv((int64_t)a->max_len * a->n_kv_heads, rows), (unsigned)(a->batch < 65535 ? a->batch : 65535));
  cudaStream_t st = (cudaStream_t)stream;
  if (a->head_dim == 128) {
    if (a->x_dtype == GL_BF16) return launch_read<128, __nv_bfloat16>(p, a->format, grid, st);
    return a->x_dtype == GL_FP16 ? launch_read<128, __half>(p, a->format, grid, st) : launch_read<128, float>(p, a->format, grid, st);
  }
  if (a->x_dtype == GL_BF16) return launch_read<64, __nv_bfloat16>(p, a->format, grid, st);
  return a->x_dtype == GL_FP16 ? launch_read<64, __half>(p, a->format, grid, st) : launch_read<64, float>(p, a->format, grid, st);
}
