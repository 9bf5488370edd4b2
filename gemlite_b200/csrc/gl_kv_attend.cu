// Attention over the quantised key/value cache for few query rows per key/value head (single tokens, small trees), the
// join of split sequences, and the entry point that picks a kernel.  sm_100a.
//
// out = softmax(c q K^T) V with K[p] = ks[p] (kq[p] - kz[p]), V[p] = vs[p] (vq[p] - vz[p]), one scale (and, in 4 bits, one zero
// point) per token and head.  The scales never touch the codes:
//   * c ks[p] multiplies the score of token p after q . kq[p];
//   * vs[p] joins the exponent: with t[p] = log2(e) c ks[p] q.kq[p] + log2 vs[p] and a running maximum M of t,
//     P[p] = 2^(t[p] - M) is the weight of the codes, and 2^(t[p] - M) / vs[p] the term of the denominator.
// So the tensor cores multiply the codes themselves, converted exactly to fp16 (e4m3, int8 and 4-bit integers are all fp16
// numbers).  q is fp16 already or is brought there from bf16 by a power of two per row (its largest channel lands in
// [1, 2): channels 2^-14 of it and smaller lose bits, at most 2^-25 of the largest each).  P carries a factor 2^15, which
// leaves the fp16 format 39 binary orders below the largest weight before a weight is lost.
#include "gl_kv.cuh"
#include "gl_kv_attend.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTinyScale = 1e-30f;
constexpr int kTile = 32;          // tokens that a warp takes at a time
constexpr int kWarps = 4;
constexpr int kStages = 3;

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Place of 16-byte chunk `c` of token row `t` in a tile of 32 rows of RB bytes.  Keys are read as one row per lane / 4 and
// consecutive chunks, values as rows 0, 2, 4, 6 (and 1, 3, .. ) and consecutive 32 / RB-chunk pieces; both orders are free of
// bank conflicts with these exchanges of chunks.
template <int RB> __device__ __forceinline__ uint32_t k_place(uint32_t t, uint32_t c) {
  if (RB == 128) return t * 128 + ((c ^ ((t & 1) << 2)) << 4);
  return t * RB + (c << 4);
}
template <int RB> __device__ __forceinline__ uint32_t v_place(uint32_t t, uint32_t c) {
  if (RB == 128) return t * 128 + ((c ^ (t & 7)) << 4);
  if (RB == 64) return (t >> 1) * 128 + (((((t & 1) << 2) + c) ^ (((t >> 1) & 3) << 1)) << 4);
  return (t >> 2) * 128 + (((((t & 3) << 1) + c) ^ ((t >> 2 & 1) << 1)) << 4);
}

template <int D, int FMT> struct Shape {
  static constexpr int RB = FMT == GL_KV_INT4 ? D / 2 : D;         // bytes of a token's row
  static constexpr int CODES = kTile * RB;
  static constexpr int K_AT = 0, V_AT = CODES, KS_AT = 2 * CODES, VS_AT = KS_AT + kTile * 4, KZ_AT = VS_AT + kTile * 4, VZ_AT = KZ_AT + kTile,
                       VALID_AT = VZ_AT + kTile, STAGE = VALID_AT + 64;
  static constexpr int LOOP = kWarps * kStages * STAGE;
};

template <int D, int FMT, int MT, typename T>
__global__ void __launch_bounds__(kWarps * 32) kv_attend_mma_kernel(const KvAttendParams p) {
  using S = Shape<D, FMT>;
  constexpr int RB = S::RB, CPT = RB / 16, NT = D / 8, KS = D / 16, ROWS = 16 * MT;
  constexpr float kShift = 15.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const KvBatch& kb = p.kb;
  gl_launch_dependents();
  gl_grid_dependency_wait();

  const int b = blockIdx.z, kvh = blockIdx.y % kb.hkv, rt_step = gridDim.y / kb.hkv;
  int first, end;
  kv_new_rows(kb, b, first, end);
  const int new_b = end - first;
  if (new_b <= 0) return;
  const int ctx = kv_len(kb, b);
  const int len = (int)min((int64_t)ctx + new_b, kv_capacity(kb));
  const int rows = new_b * p.group;
  const int chunk = kv_attend_chunk(p, len);
  const int c0 = blockIdx.x * chunk;

  uint8_t* ring = smem + warp * kStages * S::STAGE;
  const uint32_t ring_u = smem_addr(ring);

  for (int rt = blockIdx.y / kb.hkv; rt * ROWS < rows; rt += rt_step) {
    const int r_base = rt * ROWS;
    const int t_hi = min(new_b - 1, (r_base + ROWS - 1) / p.group);
    const int c1 = min(min(c0 + chunk, len), p.mask == nullptr ? ctx + t_hi + 1 : len);

    // ---- queries as the A operand, channels in the order in which the codes come out of their words
    uint32_t qa[MT][KS][4];
    float qs[MT][2];
    int q_tok[MT][2];                                     // which new token the row belongs to
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = r_base + m * 16 + g + hf * 8;
        const bool live = r < rows;
        const int t = live ? r / p.group : 0, head = kvh * p.group + (live ? r - t * p.group : 0);
        q_tok[m][hf] = t;
        const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(first + t) * p.q_sn + (int64_t)head * p.q_sh;
        uint32_t w[D / 8];                                // this lane's D / 4 channels
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          // 8-bit rows: chunks c and c + 4 of 16 channels; 4-bit rows: one piece of D / 4 channels
          const int at = FMT == GL_KV_INT4 ? c * (D / 4) + i * 8 : (i >> 1) * 64 + c * 16 + (i & 1) * 8;
          uint4 u = make_uint4(0, 0, 0, 0);
          if (live) u = *reinterpret_cast<const uint4*>(src + at);
          w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
        float factor = 1.f;
        if constexpr (sizeof(T) == 2 && !IsHalf<T>::value) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int ex = min(max((int)(top >> 7), 1), 253);
          const float inv = __int_as_float((254 - ex) << 23);
          factor = __int_as_float(ex << 23);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const __half2 h = __floats2half2_rn(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        qs[m][hf] = p.scale_log2 * factor;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          if (FMT == GL_KV_INT4) {
            const int i4 = (j >> 1) * 4;                  // words of channels 8 (j / 2) ..: (0,1) (2,3) (4,5) (6,7)
            qa[m][j][hf] = prmt(w[i4 + (j & 1)], w[i4 + 2 + (j & 1)], 0x5410);
            qa[m][j][2 + hf] = prmt(w[i4 + (j & 1)], w[i4 + 2 + (j & 1)], 0x7632);
          } else {
            qa[m][j][hf] = w[2 * j];
            qa[m][j][2 + hf] = w[2 * j + 1];
          }
        }
      }

    float o[MT][NT][4], mx[MT][2], sum[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][i][e] = 0.f;
      mx[m][0] = mx[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
    }

    const int tiles = c1 > c0 ? (c1 - c0 + kTile - 1) / kTile : 0;
    const int mine = (tiles - warp + kWarps - 1) / kWarps;              // tiles warp, warp + 4, ..

    auto slot_of = [&](int i) -> int64_t {                              // lane's token of the warp's i-th tile
      const int pos = c0 + (warp + i * kWarps) * kTile + lane;
      if (i >= mine || pos >= c1) return -1;
      const int pi = p.page_shift >= 0 ? pos >> p.page_shift : pos / kb.page_size;
      const int page = kb.page_table[b * kb.pt_stride + pi];
      if ((unsigned)page >= (unsigned)kb.num_pages) return -1;
      return ((int64_t)page * kb.hkv + kvh) * kb.page_size + (pos - pi * kb.page_size);
    };
    int64_t slot_next = slot_of(0);
    uint32_t z_pend = 0;
    int z_stage = -1;
    auto put_zeros = [&]() {
      if (FMT == GL_KV_INT4 && z_stage >= 0) {
        ring[z_stage * S::STAGE + S::KZ_AT + lane] = (uint8_t)z_pend;
        ring[z_stage * S::STAGE + S::VZ_AT + lane] = (uint8_t)(z_pend >> 8);
        z_stage = -1;
      }
    };
    auto issue = [&](int i) {
      put_zeros();
      if (i < mine) {
        const int st = i % kStages;
        const uint32_t at = ring_u + st * S::STAGE;
        const int64_t slot = slot_next;
        slot_next = slot_of(i + 1);
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
          const int t = lane / CPT + k * (32 / CPT), ch = lane % CPT;
          const int64_t s = __shfl_sync(0xffffffffu, slot, t);
          const int64_t off = s < 0 ? 0 : s * RB + ch * 16;
          cp_async16(at + S::K_AT + k_place<RB>(t, ch), p.k_codes + off, s >= 0);
          cp_async16(at + S::V_AT + v_place<RB>(t, ch), p.v_codes + off, s >= 0);
        }
        const int64_t so = slot < 0 ? 0 : slot;
        cp_async4(at + S::KS_AT + lane * 4, p.k_scales + so, slot >= 0);
        cp_async4(at + S::VS_AT + lane * 4, p.v_scales + so, slot >= 0);
        if (FMT == GL_KV_INT4) {
          z_pend = slot >= 0 ? (uint32_t)p.k_zeros[so] | (uint32_t)p.v_zeros[so] << 8 : 0u;
          z_stage = st;
        }
        const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0);
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + st * S::STAGE + S::VALID_AT) = there;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    for (int i = 0; i < mine; ++i) {
      issue(i + kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      uint8_t* st = ring + (i % kStages) * S::STAGE;
      const int tile0 = c0 + (warp + i * kWarps) * kTile;
      const uint32_t there = *reinterpret_cast<const uint32_t*>(st + S::VALID_AT);
      const bool whole = there == 0xffffffffu && tile0 + kTile <= ctx;
      // Rows of values that the sums cannot take as they are, lane = token.  A scale of (about) zero: log2 would leave no
      // denominator, so the codes become zeros under a scale that does.  e4m3's NaN among new tokens: 0 * NaN would reach
      // rows that do not see the token, so its codes become zeros under the scale NaN, which only reaches rows that do.
      const float vs_lane = *reinterpret_cast<const float*>(st + S::VS_AT + lane * 4);
      if (__any_sync(0xffffffffu, vs_lane < kTinyScale || (FMT == GL_KV_FP8 && !whole))) {
        bool nan = false;
        if (FMT == GL_KV_FP8 && !whole) {
          for (int ch = 0; ch < CPT; ++ch) {
            const uint4 u = *reinterpret_cast<const uint4*>(st + S::V_AT + v_place<RB>(lane, ch));
            const uint32_t m = 0x7f7f7f7fu, one = 0x01010101u;
            nan |= ((((u.x & m) + one) | ((u.y & m) + one) | ((u.z & m) + one) | ((u.w & m) + one)) & 0x80808080u) != 0;
          }
        }
        if (nan || vs_lane < kTinyScale) {
          for (int ch = 0; ch < CPT; ++ch) *reinterpret_cast<uint4*>(st + S::V_AT + v_place<RB>(lane, ch)) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<float*>(st + S::VS_AT + lane * 4) = nan ? __int_as_float(0x7fc00000) : kTinyScale;
          if (FMT == GL_KV_INT4) st[S::VZ_AT + lane] = 0;
        }
        __syncwarp();
      }

      // ---- scores
      float s[MT][4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][nt][e] = 0.f;
        const int t = nt * 8 + g;
        uint32_t kw[RB / 16];
        if constexpr (RB == 128) {
          *reinterpret_cast<uint4*>(kw) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c));
          *reinterpret_cast<uint4*>(kw + 4) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c + 4));
        } else if constexpr (RB == 64) {
          *reinterpret_cast<uint4*>(kw) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c));
        } else {
          *reinterpret_cast<uint2*>(kw) = *reinterpret_cast<const uint2*>(st + S::K_AT + t * RB + c * 8);
        }
        uint32_t zk = 0;
        if (FMT == GL_KV_INT4) {
          zk = 0x6400u + st[S::KZ_AT + t];
          zk |= zk << 16;
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          uint32_t b0, b1;
          if (FMT == GL_KV_INT4) {
            const uint32_t w = kw[j >> 1] >> ((j & 1) * 8);
            b0 = kv_nibbles(w, zk);
            b1 = kv_nibbles(w >> 4, zk);
          } else {
            kv_bytes<FMT>(kw[j], b0, b1);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) mma16816(s[m][nt], qa[m][j], b0, b1);
        }
      }

      // ---- exponents
      float rv[4][2];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        const float2 ks = *reinterpret_cast<const float2*>(st + S::KS_AT + (nt * 8 + 2 * c) * 4);
        const float2 vs = *reinterpret_cast<const float2*>(st + S::VS_AT + (nt * 8 + 2 * c) * 4);
        const float lx = __log2f(vs.x), ly = __log2f(vs.y);
        rv[nt][0] = __frcp_rn(vs.x);
        rv[nt][1] = __frcp_rn(vs.y);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          s[m][nt][0] = fmaf(s[m][nt][0] * ks.x, qs[m][0], lx);
          s[m][nt][1] = fmaf(s[m][nt][1] * ks.y, qs[m][0], ly);
          s[m][nt][2] = fmaf(s[m][nt][2] * ks.x, qs[m][1], lx);
          s[m][nt][3] = fmaf(s[m][nt][3] * ks.y, qs[m][1], ly);
        }
      }
      if (!whole) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = nt * 8 + 2 * c + (e & 1), at = tile0 + t - ctx;     // >= 0: which new token
              bool sees = (there >> t) & 1u;
              if (at >= 0) {
                const int own = q_tok[m][e >> 1];
                sees = sees && (p.mask == nullptr ? at <= own : at < p.mask_cols && p.mask[(int64_t)(first + own) * p.mask_stride + at] != 0);
              }
              if (!sees) s[m][nt][e] = -INFINITY;
            }
      }
      uint32_t pa[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float top[2] = {mx[m][0], mx[m][1]};
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          top[0] = fmaxf(top[0], fmaxf(s[m][nt][0], s[m][nt][1]));
          top[1] = fmaxf(top[1], fmaxf(s[m][nt][2], s[m][nt][3]));
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
          top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > mx[m][0] || top[1] > mx[m][1])) {
          const float f0 = mx[m][0] == top[0] ? 1.f : kv_exp2(mx[m][0] - top[0]), f1 = mx[m][1] == top[1] ? 1.f : kv_exp2(mx[m][1] - top[1]);
          sum[m][0] *= f0;
          sum[m][1] *= f1;
#pragma unroll
          for (int n = 0; n < NT; ++n) { o[m][n][0] *= f0; o[m][n][1] *= f0; o[m][n][2] *= f1; o[m][n][3] *= f1; }
          mx[m][0] = top[0];
          mx[m][1] = top[1];
        }
        const float sub0 = top[0] == -INFINITY ? 0.f : top[0] - kShift, sub1 = top[1] == -INFINITY ? 0.f : top[1] - kShift;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          const float e0 = kv_exp2(s[m][nt][0] - sub0), e1 = kv_exp2(s[m][nt][1] - sub0), e2 = kv_exp2(s[m][nt][2] - sub1), e3 = kv_exp2(s[m][nt][3] - sub1);
          // a token that is not seen has the weight 0, also where its scale is NaN
          sum[m][0] += (whole || s[m][nt][0] != -INFINITY ? e0 * rv[nt][0] : 0.f) + (whole || s[m][nt][1] != -INFINITY ? e1 * rv[nt][1] : 0.f);
          sum[m][1] += (whole || s[m][nt][2] != -INFINITY ? e2 * rv[nt][0] : 0.f) + (whole || s[m][nt][3] != -INFINITY ? e3 * rv[nt][1] : 0.f);
          const __half2 lo = __floats2half2_rn(e0, e1), hi = __floats2half2_rn(e2, e3);
          pa[m][nt >> 1][(nt & 1) * 2] = *reinterpret_cast<const uint32_t*>(&lo);
          pa[m][nt >> 1][(nt & 1) * 2 + 1] = *reinterpret_cast<const uint32_t*>(&hi);
        }
      }

      // ---- weighted codes: column n of the B operand's tile i is channel NT n + i
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        constexpr int VW = RB / 32;                        // words of a token's row that this lane takes
        uint32_t vw[4][VW];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int t = kk * 16 + 2 * c + (q4 & 1) + (q4 >> 1) * 8;
          if constexpr (RB == 128) *reinterpret_cast<uint4*>(vw[q4]) = *reinterpret_cast<const uint4*>(st + S::V_AT + v_place<RB>(t, g));
          else if constexpr (RB == 64) *reinterpret_cast<uint2*>(vw[q4]) = *reinterpret_cast<const uint2*>(st + S::V_AT + v_place<RB>(t, g >> 1) + (g & 1) * 8);
          else vw[q4][0] = *reinterpret_cast<const uint32_t*>(st + S::V_AT + v_place<RB>(t, g >> 2) + (g & 3) * 4);
        }
        uint32_t z0 = 0, z1 = 0;
        if (FMT == GL_KV_INT4) {
          const uint8_t* z = st + S::VZ_AT + kk * 16 + 2 * c;
          z0 = (0x6400u + z[0]) | (0x6400u + z[1]) << 16;
          z1 = (0x6400u + z[8]) | (0x6400u + z[9]) << 16;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if (FMT == GL_KV_INT4) {
              const uint32_t x = prmt(vw[0][w], vw[1][w], hf ? 0x7632 : 0x5410), y = prmt(vw[2][w], vw[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const uint32_t b0 = kv_nibbles(x >> (4 * n), z0), b1 = kv_nibbles(y >> (4 * n), z1);
#pragma unroll
                for (int m = 0; m < MT; ++m) mma16816(o[m][8 * w + 4 * hf + n], pa[m][kk], b0, b1);
              }
            } else {
              uint32_t b0[2], b1[2];
              kv_bytes<FMT>(prmt(vw[0][w], vw[1][w], hf ? 0x7362 : 0x5140), b0[0], b0[1]);
              kv_bytes<FMT>(prmt(vw[2][w], vw[3][w], hf ? 0x7362 : 0x5140), b1[0], b1[1]);
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) mma16816(o[m][4 * w + 2 * hf + n], pa[m][kk], b0[n], b1[n]);
            }
          }
        }
      }
      __syncwarp();                                        // the stage may be overwritten
    }

    // ---- the warps' parts become one: each scales its own to the common maximum
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        sum[m][hf] += __shfl_xor_sync(0xffffffffu, sum[m][hf], 1);
        sum[m][hf] += __shfl_xor_sync(0xffffffffu, sum[m][hf], 2);
      }
    __syncthreads();                                       // every warp is through with its ring
    float* part = reinterpret_cast<float*>(smem);          // [warps][ROWS][D]
    float2* ml = reinterpret_cast<float2*>(part + kWarps * ROWS * D);    // [warps][ROWS]
    if (c == 0)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) ml[warp * ROWS + m * 16 + g + hf * 8] = make_float2(mx[m][hf], sum[m][hf]);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = m * 16 + g + hf * 8;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
        const float f = mx[m][hf] == -INFINITY ? 0.f : kv_exp2(mx[m][hf] - top);
        float* dst = part + (warp * ROWS + r) * D + 2 * c * NT;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < NT; i += 4)
            *reinterpret_cast<float4*>(dst + e * NT + i) = make_float4(o[m][i][2 * hf + e] * f, o[m][i + 1][2 * hf + e] * f, o[m][i + 2][2 * hf + e] * f, o[m][i + 3][2 * hf + e] * f);
      }
    __syncthreads();
    for (int at = tid * 4; at < ROWS * D; at += kWarps * 32 * 4) {
      const int r = at / D, d = at % D;
      if (r_base + r >= rows) break;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(part + (w * ROWS + r) * D + d);
        acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
        const float2 m2 = ml[w * ROWS + r];
        l += m2.x == -INFINITY ? 0.f : m2.y * kv_exp2(m2.x - top);
      }
      const int rr = r_base + r, t = rr / p.group;
      const int64_t row = (int64_t)(first + t) * p.hq + kvh * p.group + (rr - t * p.group);
      if (p.splits > 1) {
        const int64_t pr = (int64_t)blockIdx.x * kb.n_tokens * p.hq + row;
        if (l != 0.f) *reinterpret_cast<float4*>(p.part_o + pr * D + d) = acc;     // (NaN is not 0)
        if (d == 0) p.part_ml[pr] = make_float2(top, l);
      } else {
        kv_store4<T>(reinterpret_cast<T*>(p.out) + row * D + d, acc, l);
      }
    }
    __syncthreads();
  }
}

// Joins the parts of a split sequence: one block per row, warp w takes splits w, w + 8, ..
template <int D, typename T>
__global__ void __launch_bounds__(256) kv_attend_join_kernel(const KvAttendParams p) {
  __shared__ float4 acc_s[8][D / 4];
  __shared__ float red[8];
  const int64_t row = blockIdx.x, rows = (int64_t)p.kb.n_tokens * p.hq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = (int)(row / p.hq);
  gl_launch_dependents();
  gl_grid_dependency_wait();
  // rows that belong to no sequence stay as they were
  if (p.kb.q_offsets != nullptr && (n < p.kb.q_offsets[0] || n >= p.kb.q_offsets[p.kb.batch])) return;

  float top = -INFINITY;
  for (int s = tid; s < p.splits; s += 256) {
    const float2 ml = p.part_ml[s * rows + row];
    if (ml.y != 0.f) top = fmaxf(top, ml.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, red[w]);
  __syncthreads();
  constexpr int V = D / 32;
  float acc[V] = {};
  float l = 0.f;
#pragma unroll 4
  for (int s = warp; s < p.splits; s += 8) {
    const float2 ml = p.part_ml[s * rows + row];
    if (ml.y == 0.f) continue;
    const float f = ml.x == -INFINITY ? ml.y : kv_exp2(ml.x - top);    // -inf with a sum: the sum is NaN
    l += ml.y * f;
    const float* src = p.part_o + (s * rows + row) * D + lane * V;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] += src[j] * f;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) reinterpret_cast<float*>(acc_s[warp])[lane * V + j] = acc[j];
  if (lane == 0) red[warp] = l;
  __syncthreads();
  if (tid < D / 4) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float4 x = acc_s[w][tid];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      l += red[w];
    }
    kv_store4<T>(reinterpret_cast<T*>(p.out) + row * D + tid * 4, a, l);
  }
}

template <int D, int FMT, int MT, typename T>
int launch_mma(const KvAttendParams& p, dim3 grid, cudaStream_t st) {
  constexpr int LOOP = Shape<D, FMT>::LOOP, JOIN = kWarps * 16 * MT * (D * 4 + 8), SMEM = LOOP > JOIN ? LOOP : JOIN;
  static bool set[64];
  int dev = 0;
  GL_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !set[dev]) {
    GL_CUDA_CHECK(cudaFuncSetAttribute(kv_attend_mma_kernel<D, FMT, MT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  GL_CUDA_CHECK(gl_launch_pdl(kv_attend_mma_kernel<D, FMT, MT, T>, grid, dim3(kWarps * 32), SMEM, st, p));
  return GL_OK;
}
template <int D, int FMT, typename T>
int launch_rows(const KvAttendParams& p, int mt, dim3 grid, cudaStream_t st) {
  return mt == 1 ? launch_mma<D, FMT, 1, T>(p, grid, st) : launch_mma<D, FMT, 2, T>(p, grid, st);
}
template <int D, typename T>
int launch_fmt(const KvAttendParams& p, int fmt, int mt, dim3 grid, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: return launch_rows<D, GL_KV_FP8, T>(p, mt, grid, st);
    case GL_KV_INT8: return launch_rows<D, GL_KV_INT8, T>(p, mt, grid, st);
    default: return launch_rows<D, GL_KV_INT4, T>(p, mt, grid, st);
  }
}
template <typename T>
int launch_mma_any(const KvAttendParams& p, int d, int fmt, int mt, dim3 grid, cudaStream_t st) {
  return d == 128 ? launch_fmt<128, T>(p, fmt, mt, grid, st) : launch_fmt<64, T>(p, fmt, mt, grid, st);
}

struct Plan {
  int mt, row_tiles, splits, chunk;
};

// How the work is cut.  Tokens are the long axis: a (sequence, kv head, row tile) gets as many splits as fill the SMs
// kWaves times over, none shorter than 128 tokens (one trip of the four warps).
Plan plan_of(const gl_kv_args* a) {
  Plan pl;
  const int group = a->n_q_heads / a->n_kv_heads;
  const int64_t max_rows = (int64_t)(a->max_new < a->n_tokens ? a->max_new : a->n_tokens) * group;
  pl.mt = max_rows <= 16 ? 1 : 2;
  int64_t tiles = gl_cdiv(max_rows, 16 * pl.mt);
  const int64_t most = 65535 / a->n_kv_heads;
  if (tiles > most) tiles = most;
  pl.row_tiles = tiles < 1 ? 1 : (int)tiles;
  const int64_t cap = (int64_t)a->max_pages * a->page_size;
  int64_t len = a->max_len < cap ? a->max_len : cap;
  if (len < 1) len = 1;
  const int64_t units = (int64_t)a->batch * a->n_kv_heads * pl.row_tiles, want = gl_cdiv((int64_t)gl_num_sms() * 2 * 4, units);
  int64_t chunk = gl_cdiv(gl_cdiv(len, want), 128) * 128;
  const int64_t splits = gl_cdiv(len, chunk);
  pl.splits = (int)(splits < 1024 ? splits : 1024);
  pl.chunk = (int)(gl_cdiv(gl_cdiv(len, pl.splits), 128) * 128);
  return pl;
}

int check_attend(const gl_kv_args* a) {
  if (int rc = gl_kv_check("gl_kv_attend", a)) return rc;
  if (a->x_dtype != GL_FP16 && a->x_dtype != GL_BF16) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: dtype %d (fp16 / bf16 only)", a->x_dtype);
  if (a->n_q_heads <= 0 || a->n_q_heads % a->n_kv_heads != 0) GL_FAIL(GL_E_INVALID, "gl_kv_attend: %d query heads over %d kv heads", a->n_q_heads, a->n_kv_heads);
  if (a->batch > 65535 || a->n_kv_heads > 65535) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: %d sequences, %d kv heads (at most 65535)", a->batch, a->n_kv_heads);
  if ((int64_t)a->n_tokens * a->n_q_heads > 0x7fffffffll) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: %d tokens of %d heads", a->n_tokens, a->n_q_heads);
  if ((int64_t)a->max_pages * a->page_size > 0x40000000ll) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: page table of %d x %d tokens (at most 2^30)", a->max_pages, a->page_size);
  return GL_OK;
}

uint64_t workspace_of(const gl_kv_args* a, const Plan& pl) {
  if (pl.splits <= 1) return 0;
  return (uint64_t)pl.splits * (uint64_t)a->n_tokens * (uint64_t)a->n_q_heads * (uint64_t)(a->head_dim * 4 + 8);
}

}  // namespace

extern "C" uint64_t gl_kv_attend_workspace_bytes(const gl_kv_args* a) {
  if (check_attend(a) != GL_OK || a->batch == 0 || a->n_tokens == 0) return 0;
  return workspace_of(a, plan_of(a));
}

extern "C" int gl_kv_attend(const gl_kv_args* a, void* stream) {
  if (int rc = check_attend(a)) return rc;
  if (a->batch == 0 || a->n_tokens == 0) return GL_OK;
  if (!a->q || !a->out || (((uintptr_t)a->q | (uintptr_t)a->out) & 15)) GL_FAIL(GL_E_INVALID, "gl_kv_attend: null or misaligned queries / output");
  if ((a->q_stride_n | a->q_stride_h) & 7) GL_FAIL(GL_E_INVALID, "gl_kv_attend: strides must be multiples of 8 elements");
  if (a->mask && a->mask_cols < 0) GL_FAIL(GL_E_INVALID, "gl_kv_attend: mask of %d columns", a->mask_cols);
  const Plan pl = plan_of(a);
  const uint64_t need = workspace_of(a, pl);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
    GL_FAIL(GL_E_WORKSPACE, "gl_kv_attend: workspace of %llu bytes (16-byte aligned) needed, got %llu", (unsigned long long)need, (unsigned long long)a->workspace_bytes);
  KvAttendParams p;
  p.kb = gl_kv_batch(a);
  p.k_codes = (const uint8_t*)a->k_codes; p.v_codes = (const uint8_t*)a->v_codes;
  p.k_scales = a->k_scales; p.v_scales = a->v_scales;
  p.k_zeros = a->k_zeros; p.v_zeros = a->v_zeros;
  p.q = a->q; p.out = a->out; p.mask = a->mask;
  p.q_sn = a->q_stride_n; p.q_sh = a->q_stride_h; p.mask_stride = a->mask_stride;
  p.mask_cols = a->mask_cols; p.hq = a->n_q_heads; p.group = a->n_q_heads / a->n_kv_heads;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.splits = pl.splits; p.chunk = pl.chunk;
  p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? __builtin_ctz((unsigned)a->page_size) : -1;
  const int64_t rows = (int64_t)a->n_tokens * a->n_q_heads;
  p.part_o = (float*)a->workspace;
  p.part_ml = need > 0 ? reinterpret_cast<float2*>(p.part_o + (int64_t)pl.splits * rows * a->head_dim) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)pl.splits, (unsigned)(a->n_kv_heads * pl.row_tiles), (unsigned)a->batch);
  const int rc = a->x_dtype == GL_BF16 ? launch_mma_any<__nv_bfloat16>(p, a->head_dim, a->format, pl.mt, grid, st)
                                       : launch_mma_any<__half>(p, a->head_dim, a->format, pl.mt, grid, st);
  if (rc != GL_OK || pl.splits == 1) return rc;
  const dim3 jg((unsigned)rows);
  if (a->head_dim == 128) {
    if (a->x_dtype == GL_BF16) GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<128, __nv_bfloat16>, jg, dim3(256), 0, st, p));
    else GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<128, __half>, jg, dim3(256), 0, st, p));
  } else {
    if (a->x_dtype == GL_BF16) GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<64, __nv_bfloat16>, jg, dim3(256), 0, st, p));
    else GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<64, __half>, jg, dim3(256), 0, st, p));
  }
  return GL_OK;
}
