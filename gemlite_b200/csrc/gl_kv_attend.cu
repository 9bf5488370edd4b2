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
//
// Bound by the cache's bytes, then by issue slots (conversion, about 500 instructions per 32 tokens of 128 channels).  32 decoding
// sequences of 500 to 16000 tokens, 64 / 8 heads of 128 in fp8 (559 MB): 100 us, 5.6 TB/s; 128 of 1000 to 8000 in fp8 (1.2 GB) 201 us,
// 6.1 TB/s, in int4 (640 MB) 246 us, 2.6 TB/s: the 4-bit conversion (shift, mask, subtract, permute) is the bound there, not the bytes.  One
// sequence of 131000 tokens, 8 / 1 heads, int8 (35 MB): 20 us, of which the tokens take 5.
#include "gl_kv_attend.cuh"
#include <mutex>

namespace {

constexpr float kLog2e = 1.4426950408889634f;
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
  static constexpr int K_AT = 0, V_AT = CODES, KS_AT = 2 * CODES, VS_AT = KS_AT + kTile * 4, RV_AT = VS_AT + kTile * 4, KZ_AT = RV_AT + kTile * 4,
                       VZ_AT = KZ_AT + kTile, VALID_AT = VZ_AT + kTile, STAGE = VALID_AT + 64;
  static constexpr int LOOP = kWarps * kStages * STAGE;
};

// Thread blocks per SM: what shared memory (8-bit rows of 128) and registers without spills let in.  32 decoding sequences of
// 64 / 8 heads of 128 in fp8: 99 us with two blocks and three stages, 105 us with three blocks and two.
constexpr int kv_mma_blocks(int d, int fmt, int nr) { return d == 64 ? (nr == 1 ? 4 : 3) : nr == 1 && fmt == GL_KV_INT4 ? 3 : 2; }

// Transposed products: S^T = K Q^T and O^T = V^T P^T, so that the tokens (keys) or the channels (values) are the 16 rows of the
// MMA and 8 query rows its columns: a single token of a group of 8 heads fills them.  NR tiles of 8 query rows.
template <int D, int FMT, int NR, typename T>
__global__ void __launch_bounds__(kWarps * 32, kv_mma_blocks(D, FMT, NR)) kv_attend_mma_kernel(const KvAttendParams p) {
  using S = Shape<D, FMT>;
  constexpr int RB = S::RB, CPT = RB / 16, NT = D / 8, KS = D / 16, ROWS = 8 * NR;
  constexpr float kShift = 15.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ KvPlaceScratch place_scratch;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const KvBatch& kb = p.kb;
  gl_launch_dependents();
  gl_grid_dependency_wait();
  KvWalk<ROWS> walk;
  walk.start(p, kv_place_of_block<ROWS, kWarps * 32>(p, blockIdx.x, place_scratch), blockIdx.x);

  uint8_t* ring = smem + warp * kStages * S::STAGE;
  const uint32_t ring_u = smem_addr(ring);

  KvPiece pc;
  KvCut cut{};
  while (walk.next(p, blockIdx.x, pc)) {
    KvWalk<ROWS>::note(cut, pc);
    const int first = pc.s.first, ctx = pc.s.ctx, rows = pc.rows, kvh = pc.head;
    const int c0 = pc.t0 * kKvTile, c1 = min(pc.t1 * kKvTile, pc.s.len);
    const int64_t pt_row = (int64_t)walk.b * kb.pt_stride;
    const int tiles = c1 > c0 ? (c1 - c0 + kTile - 1) / kTile : 0;
    const int mine = (tiles - warp + kWarps - 1) / kWarps;              // tiles warp, warp + 4, ..

    // ---- tokens of a tile into shared memory, kStages - 1 tiles ahead
    int page_next = -1, place_next = 0;                                 // lane's token of the tile that is issued next: its
    auto look_up = [&](int i) {                                         // page number is not touched before then
      const int pos = c0 + (warp + i * kWarps) * kTile + lane;
      page_next = -1;
      if (i < mine && pos < c1) {
        const int pi = p.page_shift >= 0 ? pos >> p.page_shift : pos / kb.page_size;
        place_next = pos - pi * kb.page_size;
        page_next = kv_load(kb.page_table + pt_row + pi);
      }
    };
    look_up(0);
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
        const uint32_t slot = kv_slot32(kb, page_next, kvh, place_next), slot0 = __shfl_sync(0xffffffffu, slot, 0);
        const bool live = slot != kNoSlot;
        look_up(i + 1);
        if (__all_sync(0xffffffffu, slot == slot0 + lane && live)) {              // 32 rows in a row: a tile inside one page
          const uint8_t *ks = p.k_codes + (int64_t)slot0 * RB + lane * 16, *vs = p.v_codes + (int64_t)slot0 * RB + lane * 16;
#pragma unroll
          for (int k = 0; k < CPT; ++k) {
            const int t = lane / CPT + k * (32 / CPT), ch = lane % CPT;
            cp_async16(at + S::K_AT + k_place<RB>(t, ch), ks + k * 512, true);
            cp_async16(at + S::V_AT + v_place<RB>(t, ch), vs + k * 512, true);
          }
        } else {
#pragma unroll
          for (int k = 0; k < CPT; ++k) {
            const int t = lane / CPT + k * (32 / CPT), ch = lane % CPT;
            const uint32_t s = __shfl_sync(0xffffffffu, slot, t);
            const int64_t off = s == kNoSlot ? 0 : (int64_t)s * RB + ch * 16;
            cp_async16(at + S::K_AT + k_place<RB>(t, ch), p.k_codes + off, s != kNoSlot);
            cp_async16(at + S::V_AT + v_place<RB>(t, ch), p.v_codes + off, s != kNoSlot);
          }
        }
        const uint32_t so = live ? slot : 0u;
        cp_async4(at + S::KS_AT + lane * 4, p.k_scales + so, live);
        cp_async4(at + S::VS_AT + lane * 4, p.v_scales + so, live);
        if (FMT == GL_KV_INT4) {
          z_pend = live ? (uint32_t)p.k_zeros[so] | (uint32_t)p.v_zeros[so] << 8 : 0u;
          z_stage = st;
        }
        const uint32_t there = __ballot_sync(0xffffffffu, live);
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + st * S::STAGE + S::VALID_AT) = there;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ---- queries as the B operand (column = row g of a tile of 8), channels in the order in which codes come out of their words
    uint32_t qb[NR][KS][2];
    float qs[NR][2];                                      // log2(e) * scale * power of two, of rows 2c and 2c + 1
    int q_tok[NR][2];                                     // their tokens
#pragma unroll
    for (int m = 0; m < NR; ++m) {
      const bool live = m * 8 + g < rows;
      const int r = pc.row0 + (live ? m * 8 + g : 0), t = r / p.group, head = kvh * p.group + (r - t * p.group);
      const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(first + t) * p.q_sn + (int64_t)head * p.q_sh;
      uint32_t w[D / 8];                                  // this lane's D / 4 channels
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        // 8-bit rows: chunks c and c + 4 of 16 channels; 4-bit rows: one piece of D / 4 channels
        const int at = FMT == GL_KV_INT4 ? c * (D / 4) + i * 8 : (i >> 1) * 64 + c * 16 + (i & 1) * 8;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (live) u = *reinterpret_cast<const uint4*>(src + at);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
      float factor = 1.f;
      if constexpr (!IsHalf<T>::value) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = min(max((int)(top >> 7), 1), 253);
        const float inv = __int_as_float((254 - ex) << 23);
        factor = __int_as_float(ex << 23);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = kv_pair<__half>(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
      }
      const float f = p.scale_log2 * factor;
#pragma unroll
      for (int e = 0; e < 2; ++e) {                       // row 2c + e is column g = 2c + e of lanes 4 g ..
        qs[m][e] = __shfl_sync(0xffffffffu, f, (2 * c + e) * 4);
        q_tok[m][e] = __shfl_sync(0xffffffffu, t, (2 * c + e) * 4);
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if (FMT == GL_KV_INT4) {
          const int i4 = (j >> 1) * 4;                    // words of channels 8 (j / 2) ..: (0,1) (2,3) (4,5) (6,7)
          qb[m][j][0] = prmt(w[i4 + (j & 1)], w[i4 + 2 + (j & 1)], 0x5410);
          qb[m][j][1] = prmt(w[i4 + (j & 1)], w[i4 + 2 + (j & 1)], 0x7632);
        } else {
          qb[m][j][0] = w[2 * j];
          qb[m][j][1] = w[2 * j + 1];
        }
      }
    }

    float o[NR][NT / 2][4], mx[NR][2], sum[NR][2];
#pragma unroll
    for (int m = 0; m < NR; ++m) {
#pragma unroll
      for (int i = 0; i < NT / 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][i][e] = 0.f;
      mx[m][0] = mx[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.f;
    }

#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      issue(i + kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      uint8_t* st = ring + (i % kStages) * S::STAGE;
      const int tile0 = c0 + (warp + i * kWarps) * kTile;
      const uint32_t there = *reinterpret_cast<const uint32_t*>(st + S::VALID_AT);
      const bool whole = there == 0xffffffffu && tile0 + kTile <= ctx;
      // Lane = token: log2 and reciprocal of its value scale.  Rows of values that the sums cannot take as they are: a scale of
      // (about) zero would leave no denominator, so the codes become zeros under a scale that does.  e4m3's NaN among new
      // tokens: 0 * NaN would reach rows that do not see the token, so its codes become zeros under the scale NaN, which only
      // reaches rows that do.
      float vs_lane = *reinterpret_cast<const float*>(st + S::VS_AT + lane * 4);
      if (__any_sync(0xffffffffu, vs_lane < kTinyScale || (FMT == GL_KV_FP8 && !whole))) {
        bool nan = false;
        if (FMT == GL_KV_FP8 && !whole) {
#pragma unroll 1
          for (int ch = 0; ch < CPT; ++ch) {
            const uint4 u = *reinterpret_cast<const uint4*>(st + S::V_AT + v_place<RB>(lane, ch));
            const uint32_t m = 0x7f7f7f7fu, one = 0x01010101u;
            nan |= ((((u.x & m) + one) | ((u.y & m) + one) | ((u.z & m) + one) | ((u.w & m) + one)) & 0x80808080u) != 0;
          }
        }
        if (nan || vs_lane < kTinyScale) {
#pragma unroll 1
          for (int ch = 0; ch < CPT; ++ch) *reinterpret_cast<uint4*>(st + S::V_AT + v_place<RB>(lane, ch)) = make_uint4(0, 0, 0, 0);
          vs_lane = nan ? __int_as_float(0x7fc00000) : kTinyScale;
          if (FMT == GL_KV_INT4) st[S::VZ_AT + lane] = 0;
        }
      }
      *reinterpret_cast<float*>(st + S::VS_AT + lane * 4) = __log2f(vs_lane);
      *reinterpret_cast<float*>(st + S::RV_AT + lane * 4) = __frcp_rn(vs_lane);
      __syncwarp();

      // ---- scores of 2 x 16 tokens: this lane's are tokens g and g + 8, rows 2c and 2c + 1
      float s[NR][2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t kw[2][RB / 16], zk[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int t = h * 16 + y * 8 + g;
          if constexpr (RB == 128) {
            *reinterpret_cast<uint4*>(kw[y]) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c));
            *reinterpret_cast<uint4*>(kw[y] + 4) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c + 4));
          } else if constexpr (RB == 64) {
            *reinterpret_cast<uint4*>(kw[y]) = *reinterpret_cast<const uint4*>(st + S::K_AT + k_place<RB>(t, c));
          } else {
            *reinterpret_cast<uint2*>(kw[y]) = *reinterpret_cast<const uint2*>(st + S::K_AT + t * RB + c * 8);
          }
          zk[y] = 0;
          if (FMT == GL_KV_INT4) zk[y] = (0x6400u + st[S::KZ_AT + t]) * 0x10001u;
        }
#pragma unroll
        for (int m = 0; m < NR; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][h][e] = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          uint32_t a[4];
          if (FMT == GL_KV_INT4) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t w = kw[y][j >> 1] >> ((j & 1) * 8);
              a[y] = kv_nibbles(w, zk[y]);
              a[2 + y] = kv_nibbles(w >> 4, zk[y]);
            }
          } else {
            kv_bytes<FMT>(kw[0][j], a[0], a[2]);
            kv_bytes<FMT>(kw[1][j], a[1], a[3]);
          }
#pragma unroll
          for (int m = 0; m < NR; ++m) mma16816(s[m][h], a, qb[m][j][0], qb[m][j][1]);
        }
      }

      // ---- exponents
      float rv[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int t = h * 16 + y * 8 + g;
          const float ks = *reinterpret_cast<const float*>(st + S::KS_AT + t * 4), lv = *reinterpret_cast<const float*>(st + S::VS_AT + t * 4);
          rv[h][y] = *reinterpret_cast<const float*>(st + S::RV_AT + t * 4);
#pragma unroll
          for (int m = 0; m < NR; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[m][h][2 * y + e] = fmaf(s[m][h][2 * y + e] * ks, qs[m][e], lv);
        }
      if (!whole) {
#pragma unroll
        for (int m = 0; m < NR; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = h * 16 + (e >> 1) * 8 + g, at = tile0 + t - ctx;     // >= 0: which new token
              bool sees = (there >> t) & 1u;
              if (at >= 0) {
                const int own = q_tok[m][e & 1];
                sees = sees && (p.mask == nullptr ? at <= own : at < p.mask_cols && p.mask[(int64_t)(first + own) * p.mask_stride + at] != 0);
              }
              if (!sees) s[m][h][e] = -INFINITY;
            }
      }
      uint32_t pb[NR][2][2];
#pragma unroll
      for (int m = 0; m < NR; ++m) {
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = fmaxf(fmaxf(s[m][0][e], s[m][0][2 + e]), fmaxf(s[m][1][e], s[m][1][2 + e]));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
          top[e] = fmaxf(fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16)), mx[m][e]);
        }
        if (__any_sync(0xffffffffu, top[0] > mx[m][0] || top[1] > mx[m][1])) {
          const float f0 = mx[m][0] == top[0] ? 1.f : kv_exp2(mx[m][0] - top[0]), f1 = mx[m][1] == top[1] ? 1.f : kv_exp2(mx[m][1] - top[1]);
          sum[m][0] *= f0;
          sum[m][1] *= f1;
#pragma unroll
          for (int n = 0; n < NT / 2; ++n) { o[m][n][0] *= f0; o[m][n][1] *= f1; o[m][n][2] *= f0; o[m][n][3] *= f1; }
          mx[m][0] = top[0];
          mx[m][1] = top[1];
        }
        const float sub[2] = {top[0] == -INFINITY ? 0.f : top[0] - kShift, top[1] == -INFINITY ? 0.f : top[1] - kShift};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float s0 = s[m][h][2 * y], s1 = s[m][h][2 * y + 1], e0 = kv_exp2(s0 - sub[0]), e1 = kv_exp2(s1 - sub[1]);
            if (whole) {
              sum[m][0] = fmaf(e0, rv[h][y], sum[m][0]);
              sum[m][1] = fmaf(e1, rv[h][y], sum[m][1]);
            } else {                                       // a token that is not seen has the weight 0, also where its scale is NaN
              sum[m][0] += s0 != -INFINITY ? e0 * rv[h][y] : 0.f;
              sum[m][1] += s1 != -INFINITY ? e1 * rv[h][y] : 0.f;
            }
            // (token g, rows 2c, 2c + 1) -> (tokens 2c, 2c + 1, row g): the B operand of the second product
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[m][h][y]) : "r"(kv_pair<__half>(e0, e1)));
          }
      }

      // ---- weighted codes: rows g and g + 8 of the A operand's tile i are channels NT g + 2 i and NT g + 2 i + 1
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        constexpr int VW = RB / 32;                        // words of a token's row that this lane takes
        uint32_t vw[4][VW];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int t = h * 16 + 2 * c + (q4 & 1) + (q4 >> 1) * 8;
          if constexpr (RB == 128) *reinterpret_cast<uint4*>(vw[q4]) = *reinterpret_cast<const uint4*>(st + S::V_AT + v_place<RB>(t, g));
          else if constexpr (RB == 64) *reinterpret_cast<uint2*>(vw[q4]) = *reinterpret_cast<const uint2*>(st + S::V_AT + v_place<RB>(t, g >> 1) + (g & 1) * 8);
          else vw[q4][0] = *reinterpret_cast<const uint32_t*>(st + S::V_AT + v_place<RB>(t, g >> 2) + (g & 3) * 4);
        }
        uint32_t z0 = 0, z1 = 0;
        if (FMT == GL_KV_INT4) {
          const uint8_t* z = st + S::VZ_AT + h * 16 + 2 * c;
          z0 = (0x6400u + z[0]) | (0x6400u + z[1]) << 16;
          z1 = (0x6400u + z[8]) | (0x6400u + z[9]) << 16;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if (FMT == GL_KV_INT4) {
              const uint32_t x = prmt(vw[0][w], vw[1][w], hf ? 0x7632 : 0x5410), y = prmt(vw[2][w], vw[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const uint32_t a[4] = {kv_nibbles(x >> (8 * n), z0), kv_nibbles(x >> (8 * n + 4), z0), kv_nibbles(y >> (8 * n), z1), kv_nibbles(y >> (8 * n + 4), z1)};
#pragma unroll
                for (int m = 0; m < NR; ++m) mma16816(o[m][4 * w + 2 * hf + n], a, pb[m][h][0], pb[m][h][1]);
              }
            } else {
              uint32_t a[4];
              kv_bytes<FMT>(prmt(vw[0][w], vw[1][w], hf ? 0x7362 : 0x5140), a[0], a[1]);
              kv_bytes<FMT>(prmt(vw[2][w], vw[3][w], hf ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
              for (int m = 0; m < NR; ++m) mma16816(o[m][2 * w + hf], a, pb[m][h][0], pb[m][h][1]);
            }
          }
      }
      __syncwarp();                                        // the stage may be overwritten
    }

    // ---- the warps' parts become one: each scales its own to the common maximum
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int m = 0; m < NR; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[m][e] += __shfl_xor_sync(0xffffffffu, sum[m][e], 4);
        sum[m][e] += __shfl_xor_sync(0xffffffffu, sum[m][e], 8);
        sum[m][e] += __shfl_xor_sync(0xffffffffu, sum[m][e], 16);
      }
    __syncthreads();                                       // every warp is through with its ring
    float* part = reinterpret_cast<float*>(smem);          // [warps][ROWS][D]
    float2* ml = reinterpret_cast<float2*>(part + kWarps * ROWS * D);    // [warps][ROWS]
    if (g == 0)
#pragma unroll
      for (int m = 0; m < NR; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) ml[warp * ROWS + m * 8 + 2 * c + e] = make_float2(mx[m][e], sum[m][e]);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < NR; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = m * 8 + 2 * c + e;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
        const float f = mx[m][e] == -INFINITY ? 0.f : kv_exp2(mx[m][e] - top);
        float* dst = part + (warp * ROWS + r) * D + NT * g;
#pragma unroll
        for (int i = 0; i < NT / 2; i += 2)
          *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[m][i][e] * f, o[m][i][2 + e] * f, o[m][i + 1][e] * f, o[m][i + 1][2 + e] * f);
      }
    __syncthreads();
    for (int at = tid * 4; at < rows * D; at += kWarps * 32 * 4) {
      const int r = at / D, d = at % D;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(part + (w * ROWS + r) * D + d);
        acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
        const float2 m2 = ml[w * ROWS + r];
        l += m2.x == -INFINITY ? (m2.y == 0.f ? 0.f : m2.y) : m2.y * kv_exp2(m2.x - top);
      }
      const int rr = pc.row0 + r, t = rr / p.group;
      if (pc.whole) {
        kv_store4<T>(reinterpret_cast<T*>(p.out) + ((int64_t)(first + t) * p.hq + kvh * p.group + (rr - t * p.group)) * D + d, acc, l);
      } else {
        const int64_t pr = (int64_t)pc.slot * ROWS + r;
        *reinterpret_cast<float4*>(p.part_o + pr * D + d) = acc;
        if (d == 0) p.part_ml[pr] = make_float2(top, l);
      }
    }
    __syncthreads();
  }
  if (tid == 0 && p.cuts != nullptr) p.cuts[blockIdx.x] = cut;
}

// Joins the parts of the units that block borders cut: blocks (i, *) look after the unit that block i began and did not
// finish.  Few parts: a warp per row; many (one long sequence): a block per row,
// warp w takes parts w, w + WARPS, ..
constexpr int kJoinMax = 1024;                 // thread blocks of a launch, at most
template <int ROWS, int D, typename T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) kv_attend_join_kernel(const KvAttendParams p) {
  __shared__ float4 acc_s[WARPS][D / 4];
  __shared__ float2 red[WARPS];
  __shared__ float weight[kJoinMax];
  __shared__ int last;
  constexpr int V = D / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  gl_launch_dependents();
  gl_grid_dependency_wait();
  // WARPS = 8: block x looks after the unit that block x of the main kernel began.  WARPS = 32, for few units: block x looks for
  // the x-th cut unit, and the x + gridDim.x-th, ..
  for (int x = blockIdx.x;; x += gridDim.x) {
    int i0 = x;
    if (WARPS == 32) {
      const bool starts = tid < p.blocks && (p.cuts[tid].flags & 1);
      const uint32_t who = __ballot_sync(0xffffffffu, starts);
      __syncthreads();
      if (tid == 0) last = -1;
      if (lane == 0) red[warp].x = __int_as_float(__popc(who));
      __syncthreads();
      int before = __popc(who & ((1u << lane) - 1u));
      for (int w = 0; w < warp; ++w) before += __float_as_int(red[w].x);
      if (starts && before == x) last = tid;
      __syncthreads();
      i0 = last;
      __syncthreads();
      if (i0 < 0) return;
    } else if (x >= p.blocks - 1) {
      return;
    }
    const KvCut cut = p.cuts[i0];
    if ((cut.flags & 1) == 0) continue;
    // the unit's last part: the first later block that finishes what it goes on with (blocks in between hold nothing else)
    if (tid == 0) last = p.blocks - 1;
    __syncthreads();
    for (int i = i0 + 1 + tid; i < p.blocks; i += WARPS * 32) {
      if (i > *(volatile int*)&last) break;
      if (p.cuts[i].flags & 4) { atomicMin(&last, i); break; }
    }
    __syncthreads();
    const int i1 = last, n = i1 - i0 + 1;
    auto part = [&](int k) { return (int64_t)(k == 0 ? 2 * i0 + 1 : 2 * (i0 + k)) * ROWS; };
    auto dst_of = [&](int r) {
      const int rr = cut.row0 + r, t = rr / p.group;
      return reinterpret_cast<T*>(p.out) + ((int64_t)(cut.first + t) * p.hq + cut.head * p.group + (rr - t * p.group)) * D;
    };
    // weight of a part: 0 where it saw nothing; a sum of NaN with the maximum -inf stays one
    auto weight_of = [&](float2 ml, float top) { return ml.y == 0.f ? 0.f : ml.x == -INFINITY ? ml.y : kv_exp2(ml.x - top); };

    if (n <= 16) {
      for (int r = blockIdx.y * WARPS + warp; r < cut.rows; r += gridDim.y * WARPS) {
        const float2 ml = lane < n ? p.part_ml[part(lane) + r] : make_float2(-INFINITY, 0.f);
        float top = ml.y != 0.f ? ml.x : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float f = weight_of(ml, top);
        float l = f == 0.f ? 0.f : ml.y * f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        float acc[V] = {};
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          float x[V];
          kv_load_n<V>(p.part_o + (part(k) + r) * D + lane * V, x);
          const float w = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += w == 0.f ? 0.f : x[j] * w;
        }
        const float q = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = l == 0.f ? 0.f : acc[j] * q;
        kv_store_n<T, V>(dst_of(r) + lane * V, acc);
      }
      continue;
    }
    for (int r = blockIdx.y; r < cut.rows; r += gridDim.y) {
      float top = -INFINITY;
      for (int k = tid; k < n; k += WARPS * 32) {
        const float2 ml = p.part_ml[part(k) + r];
        if (ml.y != 0.f) top = fmaxf(top, ml.x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) red[warp].x = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[w].x);
      float l = 0.f;
      for (int k = tid; k < n; k += WARPS * 32) {
        const float2 ml = p.part_ml[part(k) + r];
        const float f = weight_of(ml, top);
        weight[k] = f;
        l += f == 0.f ? 0.f : ml.y * f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane == 0) red[warp].y = l;
      __syncthreads();
      float acc[V] = {};
#pragma unroll 8
      for (int k = warp; k < n; k += WARPS) {
        float x[V];
        kv_load_n<V>(p.part_o + (part(k) + r) * D + lane * V, x);
        const float w = weight[k];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += w == 0.f ? 0.f : x[j] * w;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) reinterpret_cast<float*>(acc_s[warp])[lane * V + j] = acc[j];
      __syncthreads();
      if (tid < D / 4) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 x = acc_s[w][tid];
          a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
          l += red[w].y;
        }
        kv_store4<T>(dst_of(r) + tid * 4, a, l);
      }
      __syncthreads();
    }
  }
}

template <int D, int FMT, int NR, typename T>
int launch_mma(const KvAttendParams& p, cudaStream_t st) {
  constexpr int LOOP = Shape<D, FMT>::LOOP, JOIN = kWarps * 8 * NR * (D * 4 + 8), SMEM = LOOP > JOIN ? LOOP : JOIN;
  if (int rc = kv_allow_smem((const void*)kv_attend_mma_kernel<D, FMT, NR, T>, SMEM)) return rc;
  GL_CUDA_CHECK(gl_launch_pdl(kv_attend_mma_kernel<D, FMT, NR, T>, dim3((unsigned)p.blocks), dim3(kWarps * 32), SMEM, st, p));
  return GL_OK;
}
template <int D, typename T>
int launch_fmt(const KvAttendParams& p, int fmt, int rows, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: return rows == 8 ? launch_mma<D, GL_KV_FP8, 1, T>(p, st) : launch_mma<D, GL_KV_FP8, 2, T>(p, st);
    case GL_KV_INT8: return rows == 8 ? launch_mma<D, GL_KV_INT8, 1, T>(p, st) : launch_mma<D, GL_KV_INT8, 2, T>(p, st);
    default: return rows == 8 ? launch_mma<D, GL_KV_INT4, 1, T>(p, st) : launch_mma<D, GL_KV_INT4, 2, T>(p, st);
  }
}
struct Plan {
  int rows, blocks, join_y;      // rows of a unit, thread blocks of the main kernel, blocks per cut unit of the join
  bool join_many;                // units are cut into many parts
  int units;                     // .. then: an upper bound of the cut units
};

template <int ROWS, int D, typename T>
int launch_join(const KvAttendParams& p, const Plan& pl, cudaStream_t st) {
  const dim3 grid((unsigned)(pl.join_many ? pl.units : p.blocks - 1), (unsigned)pl.join_y);
  if (pl.join_many) GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<ROWS, D, T, 32>, grid, dim3(1024), 0, st, p));
  else GL_CUDA_CHECK(gl_launch_pdl(kv_attend_join_kernel<ROWS, D, T, 8>, grid, dim3(256), 0, st, p));
  return GL_OK;
}

template <int D, typename T>
int launch_all(const KvAttendParams& p, const gl_kv_args* a, const Plan& pl, cudaStream_t st) {
  if (int rc = pl.rows == kKvTcRows ? gl_kv_attend_tc_launch(p, D, a->format, a->x_dtype, st) : launch_fmt<D, T>(p, a->format, pl.rows, st)) return rc;
  if (p.blocks == 1) return GL_OK;
  if (pl.rows == kKvTcRows) return launch_join<kKvTcRows, D, T>(p, pl, st);
  return pl.rows == 8 ? launch_join<8, D, T>(p, pl, st) : launch_join<16, D, T>(p, pl, st);
}

// Few rows per kv head: the mma.sync kernel, which holds 8 or 16 rows in registers; more: the tcgen05 kernel with 256 (one block per SM).
// 64 sequences of 500 to 4000 tokens, 8 kv heads of 128, us by mma.sync / tcgen05 at so many rows per kv head:
//   fp8   8: 61 / 219   16: 83 / 230   24: 149 / 232   32: 154 / 233   40: 221 / 235   48: 228 / 240   64: 296 / 246   128: 591 / 279
//   int4  8: 74 / 198   16: 106 / 208  24: 190 / 211   32: 193 / 214   40: 274 / 218   48: 280 / 223   64: 366 / 226   128: 713 / 260
// Up to 32 rows (two passes over the codes) the first is faster in every format and head size; behind it 4 bits want the second, 8 bits
// lose 6 % at 40 rows and gain 20 % at 64.
Plan plan_of(const gl_kv_args* a) {
  Plan pl;
  const int group = a->n_q_heads / a->n_kv_heads;
  int64_t max_rows = (int64_t)(a->max_new < a->n_tokens ? a->max_new : a->n_tokens) * group;
  if (max_rows < 1) max_rows = 1;
  const bool tc = a->kernel_override == 2 || (a->kernel_override == 0 && max_rows > 32);
  pl.rows = tc ? kKvTcRows : max_rows <= 8 ? 8 : 16;
  const int live_rows = (int)(max_rows < pl.rows ? max_rows : pl.rows);
  const int64_t cap = (int64_t)a->max_pages * a->page_size;
  int64_t len = a->max_len < cap ? a->max_len : cap;
  if (len < 1) len = 1;
  const int64_t units = (int64_t)a->batch * a->n_kv_heads * gl_cdiv(max_rows, pl.rows), work = units * gl_cdiv(len, kKvTile);
  int64_t most = (int64_t)gl_num_sms() * (tc ? 1 : kv_mma_blocks(a->head_dim, a->format, pl.rows / 8));
  if (most > kJoinMax) most = kJoinMax;
  pl.blocks = (int)(work < most ? work : most);
  // units cut into many parts are joined by a block per row, others by one per 8 rows
  pl.join_many = pl.blocks > 16 * units;
  pl.units = pl.join_many ? (int)units : 0;
  const int y = pl.join_many ? live_rows : (live_rows + 7) / 8;
  pl.join_y = y < 16 ? y : 16;
  return pl;
}

int check_attend(const gl_kv_args* a) {
  if (int rc = gl_kv_check("gl_kv_attend", a)) return rc;
  if (a->x_dtype != GL_FP16 && a->x_dtype != GL_BF16) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: dtype %d (fp16 / bf16 only)", a->x_dtype);
  if (a->n_q_heads <= 0 || a->n_q_heads % a->n_kv_heads != 0) GL_FAIL(GL_E_INVALID, "gl_kv_attend: %d query heads over %d kv heads", a->n_q_heads, a->n_kv_heads);
  if (a->kernel_override < 0 || a->kernel_override > 2) GL_FAIL(GL_E_INVALID, "gl_kv_attend: kernel_override %d", a->kernel_override);
  // row numbers and tile counts of a sequence stay below 2^31, tiles in all times blocks below 2^63
  if ((int64_t)a->n_tokens * a->n_q_heads > 0x7fffffffll) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: %d tokens of %d heads", a->n_tokens, a->n_q_heads);
  if ((int64_t)a->max_pages * a->page_size > 0x40000000ll) GL_FAIL(GL_E_UNSUPPORTED, "gl_kv_attend: page table of %d x %d tokens (at most 2^30)", a->max_pages, a->page_size);
  return GL_OK;
}

uint64_t workspace_of(const gl_kv_args* a, const Plan& pl) {
  if (pl.blocks <= 1) return 0;
  return (uint64_t)pl.blocks * (2ull * (uint64_t)pl.rows * (uint64_t)(a->head_dim * 4 + 8) + sizeof(KvCut));
}

}  // namespace

int kv_allow_smem(const void* kernel, int bytes) {
  // remembered per kernel and device; without room left the attribute is set every time, which does no harm
  struct Entry { const void* kernel; int dev; };
  static Entry done[512];
  static int count = 0;
  static std::mutex mu;
  int dev = 0;
  GL_CUDA_CHECK(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < count; ++i)
    if (done[i].kernel == kernel && done[i].dev == dev) return GL_OK;
  GL_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (count < 512) done[count++] = Entry{kernel, dev};
  return GL_OK;
}

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
  p.blocks = pl.blocks;
  p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? __builtin_ctz((unsigned)a->page_size) : -1;
  p.part_o = (float*)a->workspace;
  p.cuts = need > 0 ? reinterpret_cast<KvCut*>((uint8_t*)a->workspace + 2ull * pl.blocks * pl.rows * (a->head_dim * 4 + 8)) : nullptr;
  p.part_ml = need > 0 ? reinterpret_cast<float2*>(p.part_o + 2ll * pl.blocks * pl.rows * a->head_dim) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->head_dim == 128)
    return a->x_dtype == GL_BF16 ? launch_all<128, __nv_bfloat16>(p, a, pl, st) : launch_all<128, __half>(p, a, pl, st);
  return a->x_dtype == GL_BF16 ? launch_all<64, __nv_bfloat16>(p, a, pl, st) : launch_all<64, __half>(p, a, pl, st);
}
