// Quantised key/value cache: write (head norms, rotary positions and quantisation in one pass) and read back, sm_100a.
//
// Both kernels move bytes: every operand is read once with 16-byte loads, every output written once.  A row (one token's
// head) is spread over head_dim / 8 lanes of 8 channels each, so that norms and maxima are three or four shuffles and the
// rotation's partner channel is one.
#include "gl_kv.cuh"

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
  int32_t hq, rot, interleaved, table_rows, norm_dtype;
  float eps;
};

// One block per token (and slice of its heads): the token's rotation, its norm weights and its slot are fetched once and
// serve all of its heads.  LPR lanes per row.  The order of the fp32 operations is the one of the formulas, without fused
// multiply-adds, and the sum of squares is kept in fp64: a code next to a rounding border then does not depend on how
// the row was spread over lanes.
// 8192 tokens of 64 + 2 x 8 heads of 128 (323 MB): see the table in the file's last comment.
template <typename T, int LPR, int FMT>
__global__ void __launch_bounds__(256) kv_write_kernel(const WriteParams p) {
  constexpr int D = LPR * 8, GROUPS = 256 / LPR;
  const int n = blockIdx.x;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const unsigned gmask = (LPR == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / LPR * LPR);
  gl_launch_dependents();
  gl_grid_dependency_wait();

  // sequence of row n: how many sequences end at or before it
  int b = 0, i = 0;
  if (p.kb.q_offsets != nullptr) {
    for (int base = 0; base < p.kb.batch; base += 256) {
      const int t = base + threadIdx.x;
      b += __syncthreads_count(t < p.kb.batch && p.kb.q_offsets[t + 1] <= n);
    }
    if (b >= p.kb.batch || n < p.kb.q_offsets[0]) return;
    i = n - p.kb.q_offsets[b];
  } else {
    const int t = p.kb.n_tokens / p.kb.batch;
    b = n / t;
    i = n - b * t;
  }
  const int64_t pos_in_seq = (int64_t)max(p.kb.lens[b], 0) + i;
  const int64_t slot0 = kv_slot(p.kb, b, 0, pos_in_seq);

  // this lane's share of the rotation: cosine and sine of its 8 channels (interleaved: 4 pairs)
  float cs[8], sn[8];
  bool bad_pos = false;
  const bool turns = lane * 8 < p.rot;
  if (p.rot > 0) {
    const int row = p.positions[n];
    bad_pos = (unsigned)row >= (unsigned)p.table_rows;
    if (turns && !bad_pos) {
      const float* t = p.cos_sin + (int64_t)row * p.rot;
      const int half = p.rot / 2;
      const int at = p.interleaved ? lane * 4 : (lane * 8 < half ? lane * 8 : lane * 8 - half);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = p.interleaved ? at + j / 2 : at + j;
        cs[j] = t[e];
        sn[j] = t[half + e];
      }
    } else if (turns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) { cs[j] = __int_as_float(0x7fc00000); sn[j] = cs[j]; }
    }
  }
  const int partner = lane * 8 < p.rot / 2 ? p.rot / 16 : -(p.rot / 16);   // in lanes

  const int hq = p.q != nullptr ? p.hq : 0, rows = hq + 2 * p.kb.hkv;
  float w[8];
  int w_of = -1;
  for (int r0 = blockIdx.y * GROUPS; r0 < rows; r0 += gridDim.y * GROUPS) {
    const int r = r0 + group;
    if (r >= rows) break;                     // whole groups leave together; the shuffles below name the group's lanes
    const int kind = r < hq ? 0 : r < hq + p.kb.hkv ? 1 : 2, h = kind == 0 ? r : kind == 1 ? r - hq : r - hq - p.kb.hkv;
    const T* src = kind == 0 ? reinterpret_cast<const T*>(p.q) + n * p.q_sn + h * p.q_sh
                 : kind == 1 ? reinterpret_cast<const T*>(p.k) + n * p.k_sn + h * p.k_sh
                             : reinterpret_cast<const T*>(p.v) + n * p.v_sn + h * p.v_sh;
    const uint4 u = *reinterpret_cast<const uint4*>(src + lane * 8);
    float x[8];
    {
      const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = Half2Of<T>::up(uw[j]);
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
    if (kind < 2) {
      const void* nw = kind == 0 ? p.q_norm : p.k_norm;
      if (nw != nullptr) {
        if (w_of != kind) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = gl_load_as_float(nw, lane * 8 + j, p.norm_dtype);
          w_of = kind;
        }
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += (double)x[j] * (double)x[j];
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o);
        const float mean = (float)(ss * (1.0 / D));
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, p.eps)));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(__fmul_rn(x[j], inv), w[j]);
      }
      if (p.rot > 0) {
        if (p.interleaved) {
          if (turns) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
              const float a = x[j], c = x[j + 1];
              x[j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(c, sn[j]));
              x[j + 1] = __fadd_rn(__fmul_rn(c, cs[j]), __fmul_rn(a, sn[j]));
            }
          }
        } else {
          const int from = (threadIdx.x & 31) + (turns ? partner : 0);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float other = __shfl_sync(gmask, x[j], from);
            if (turns) {
              const float own = __fmul_rn(x[j], cs[j]), turn = __fmul_rn(other, sn[j]);
              x[j] = partner > 0 ? __fsub_rn(own, turn) : __fadd_rn(own, turn);
            }
          }
        }
        if (bad_pos) {                        // channels that do not turn as well: no half-valid rows
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = __int_as_float(0x7fc00000);
        }
      }
    }
    if (kind == 0) {
      uint4 o;
      o.x = Half2Of<T>::down(x[0], x[1]);
      o.y = Half2Of<T>::down(x[2], x[3]);
      o.z = Half2Of<T>::down(x[4], x[5]);
      o.w = Half2Of<T>::down(x[6], x[7]);
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.q_out) + ((int64_t)n * p.hq + h) * D + lane * 8) = o;
      continue;
    }
    if (slot0 < 0) continue;
    const int which = kind - 1;
    const int64_t slot = slot0 + (int64_t)h * p.kb.page_size;
    // |x| as integers: infinities and NaN are the largest
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(gmask, top, o));
    const bool finite = top < 0x7f800000u;
    if (FMT == GL_KV_INT4) {
      float lo = 0.f, hi = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) { lo = fminf(lo, x[j]); hi = fmaxf(hi, x[j]); }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(gmask, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(gmask, hi, o));
      }
      const float scale = fmaxf(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 1e-6f);
      const float zero = fminf(fmaxf(rintf(__fdiv_rn(-lo, scale)), 0.f), 15.f);
      uint32_t o = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(x[j], scale)) + zero, 0.f), 15.f);
        o |= (uint32_t)(int)c << (4 * j);
      }
      reinterpret_cast<uint32_t*>(p.codes[which] + slot * (D / 2))[lane] = finite ? o : 0u;
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
        const float c = fminf(fmaxf(__fdiv_rn(x[j], scale), -qmax), qmax);
        const uint32_t byte = FMT == GL_KV_FP8 ? (uint32_t)__nv_cvt_float_to_fp8(c, __NV_SATFINITE, __NV_E4M3) : (uint32_t)(uint8_t)(int8_t)(int)rintf(c);
        o[j >> 2] |= byte << (8 * (j & 3));
      }
      reinterpret_cast<uint2*>(p.codes[which] + slot * D)[lane] = finite ? make_uint2(o[0], o[1]) : make_uint2(0u, 0u);
      if (lane == 0) p.scales[which][slot] = finite ? scale : __int_as_float(0x7fc00000);
    }
  }
}

struct ReadParams {
  KvBatch kb;
  const uint8_t *codes[2], *zeros[2];
  const float* scales[2];
  void* out[2];
  int32_t max_len, out_dtype;
};

// One lane per 16 channels of a row, keys and values of the same slot by the same lane.
template <int D, int FMT, typename O>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p) {
  constexpr int LPR = D / 16, ROWS = 256 / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  const int h = blockIdx.y;
  gl_launch_dependents();
  gl_grid_dependency_wait();
  if (t >= p.max_len) return;
  for (int b = blockIdx.z; b < p.kb.batch; b += gridDim.z) {
    const int64_t slot = t < p.kb.lens[b] ? kv_slot(p.kb, b, h, t) : -1;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[16];
      if (slot >= 0) {
        const float scale = p.scales[w][slot];
        if (FMT == GL_KV_INT4) {
          const uint2 u = *reinterpret_cast<const uint2*>(p.codes[w] + slot * (D / 2) + lane * 8);
          const int zero = p.zeros[w][slot];
          const uint32_t uw[2] = {u.x, u.y};
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = (float)((int)((uw[j >> 3] >> (4 * (j & 7))) & 15u) - zero) * scale;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(p.codes[w] + slot * D + lane * 16);
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t byte = (uw[j >> 2] >> (8 * (j & 3))) & 255u;
            x[j] = (FMT == GL_KV_FP8 ? gl_e4m3_to_float(byte) : (float)(int8_t)byte) * scale;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.f;
      }
      O* dst = reinterpret_cast<O*>(p.out[w]) + (((int64_t)b * p.max_len + t) * p.kb.hkv + h) * D + lane * 16;
      if constexpr (sizeof(O) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(dst)[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
      } else {
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = Half2Of<O>::down(x[2 * j], x[2 * j + 1]);
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
}

template <typename T, int LPR>
int launch_write(const WriteParams& p, int fmt, dim3 grid, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_FP8>, grid, dim3(256), 0, st, p)); break;
    case GL_KV_INT8: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_INT8>, grid, dim3(256), 0, st, p)); break;
    default: GL_CUDA_CHECK(gl_launch_pdl(kv_write_kernel<T, LPR, GL_KV_INT4>, grid, dim3(256), 0, st, p)); break;
  }
  return GL_OK;
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
  if ((a->q_norm || a->k_norm) && a->norm_dtype != GL_FP32 && a->norm_dtype != GL_FP16 && a->norm_dtype != GL_BF16)
    GL_FAIL(GL_E_INVALID, "gl_kv_write: norm weights of dtype %d", a->norm_dtype);
  WriteParams p;
  p.kb = gl_kv_batch(a);
  p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->out;
  p.q_norm = a->q_norm; p.k_norm = a->k_norm; p.cos_sin = a->cos_sin; p.positions = a->positions;
  p.codes[0] = (uint8_t*)a->k_codes; p.codes[1] = (uint8_t*)a->v_codes;
  p.zeros[0] = a->k_zeros; p.zeros[1] = a->v_zeros;
  p.scales[0] = a->k_scales; p.scales[1] = a->v_scales;
  p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h; p.k_sn = a->k_stride_n; p.k_sh = a->k_stride_h; p.v_sn = a->v_stride_n; p.v_sh = a->v_stride_h;
  p.hq = a->n_q_heads; p.rot = a->rot_dim; p.interleaved = a->interleaved; p.table_rows = a->table_rows; p.norm_dtype = a->norm_dtype;
  p.eps = a->eps;
  // few tokens: their heads are spread over blocks until every SM has a few; many: one block walks a token's heads
  const int lpr = a->head_dim / 8, groups = 256 / lpr;
  const int64_t slices = gl_cdiv((a->q ? a->n_q_heads : 0) + 2 * a->n_kv_heads, groups), want = gl_cdiv((int64_t)gl_num_sms() * 8, a->n_tokens);
  const dim3 grid((unsigned)a->n_tokens, (unsigned)(slices < want ? slices : want));
  cudaStream_t st = (cudaStream_t)stream;
  if (a->x_dtype == GL_BF16)
    return lpr == 16 ? launch_write<__nv_bfloat16, 16>(p, a->format, grid, st) : launch_write<__nv_bfloat16, 8>(p, a->format, grid, st);
  return lpr == 16 ? launch_write<__half, 16>(p, a->format, grid, st) : launch_write<__half, 8>(p, a->format, grid, st);
}

extern "C" int gl_kv_read(const gl_kv_args* a, void* stream) {
  if (int rc = gl_kv_check("gl_kv_read", a)) return rc;
  if (a->x_dtype != GL_FP16 && a->x_dtype != GL_BF16 && a->x_dtype != GL_FP32) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_read: output dtype %d", a->x_dtype);
  if (a->batch == 0 || a->max_len == 0) return GL_OK;
  if (!a->out || !a->out_v || (((uintptr_t)a->out | (uintptr_t)a->out_v) & 15)) GL_FAIL(GL_E_INVALID, "gl_kv_read: null or misaligned output");
  if (a->n_kv_heads > 65535) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_read: %d heads", a->n_kv_heads);
  ReadParams p;
  p.kb = gl_kv_batch(a);
  p.codes[0] = (const uint8_t*)a->k_codes; p.codes[1] = (const uint8_t*)a->v_codes;
  p.zeros[0] = a->k_zeros; p.zeros[1] = a->v_zeros;
  p.scales[0] = a->k_scales; p.scales[1] = a->v_scales;
  p.out[0] = a->out; p.out[1] = a->out_v;
  p.max_len = a->max_len; p.out_dtype = a->x_dtype;
  const int rows = 256 / (a->head_dim / 16);
  const dim3 grid((unsigned)gl_cdiv(a->max_len, rows), (unsigned)a->n_kv_heads, (unsigned)(a->batch < 65535 ? a->batch : 65535));
  cudaStream_t st = (cudaStream_t)stream;
  if (a->head_dim == 128) {
    if (a->x_dtype == GL_BF16) return launch_read<128, __nv_bfloat16>(p, a->format, grid, st);
    return a->x_dtype == GL_FP16 ? launch_read<128, __half>(p, a->format, grid, st) : launch_read<128, float>(p, a->format, grid, st);
  }
  if (a->x_dtype == GL_BF16) return launch_read<64, __nv_bfloat16>(p, a->format, grid, st);
  return a->x_dtype == GL_FP16 ? launch_read<64, __half>(p, a->format, grid, st) : launch_read<64, float>(p, a->format, grid, st);
}
