// Attention over the quantised key/value cache for many query rows per kv head (trees of drafted tokens, prompt chunks) on
// tcgen05, sm_100a.
//
// The mathematics is that of gl_kv_attend.cu.  With 128 rows a score costs more than a code, so the scales go into the codes
// where that is safe: per 32 tokens, with KS and VS powers of two set by their largest scales,
//   K'[p] = fp16(kq[p] ks[p] / KS),  V'[p] = fp16(vq[p] vs[p] / VS)          (one rounding of 2^-11 each; codes are exact)
//   S = q K'^T,  P = 2^(a S + log2 VS - M + 7),  O += P V',  l += sum P / VS,  a = log2(e) c KS (times q's power of two)
// and a score costs one multiply-add, one exponential, one maximum and one addition.  None of these numbers is a subnormal
// fp16 number as long as the scales lie near each other (kSpread, kSpreadV), so the choice of KS and VS changes no bit.  Where
// they lie further apart, and in tiles that some row of the unit does not see all of (new tokens under a mask; without one those
// behind the first row's own: a token that a row does not see must not round what it sees), K' or V' stay the codes, and ks[p],
// or log2 vs[p] and 1 / vs[p], go to the scores, as in the other kernel.
// M is a maximum of the exponents that lags: it is raised, and O and l are scaled, only when a row's new maximum is more than
// 2^8 above it (P stays below 2^15 then, fp16's range, and keeps 31 binary orders below M).  Each row decides for itself: what its
// neighbours see does not reach its roundings.
//
// One persistent block per SM, 17 working warps:
//   warps 0-3, 4-7    two streams of 128 rows: scores out of TMEM, weights back into TMEM (over the scores), rescaling, output
//   warps 8-11, 12-15 keys and values: codes from global memory (a tile ahead, in registers), conversion, swizzled shared
//                     memory (2 stages each); a warp takes 32 tokens of every tile
//   warp 16           one lane issues tcgen05.mma: S (operands in shared memory) and O (weights in TMEM, values MN-major)
// While one stream's warps exponentiate, the tensor cores work on the other.  A unit with more than 128 live rows gives each
// stream half of them, and both use every tile; with fewer, both streams hold the same rows and take every other tile, and
// stream 1 hands its part to stream 0 at the end.
//
// Bound by a stream's chain (scores, two passes over them, weights, products): a tile of 128 tokens takes about 7000 cycles where
// the tensor pipe and the exponentials need about 2050 each.  8 trees of 64 tokens over 7000 to 16000, 64 / 8 heads of 128 in fp8
// (193 GFLOP): 327 us, 591 TFLOP/s; 1000 tokens over 7000 (246 GFLOP): 400 us, 614 TFLOP/s.  The compiler spills 268 bytes for heads of 128
// and 84 for heads of 64, the same in every format and type.
#include "gl_kv_attend.cuh"
#include "gl_tc_common.cuh"

namespace {
using namespace gltc;

// 0, or what waits that gave up left since it was last cleared: 1 a wait of the roles, 2 the one before the TMEM goes back
__device__ int g_wait_status;

constexpr int kThreads = 20 * 32;             // 17 warps work; 20 fill the five warp groups that share out the registers
constexpr int kMeta = 4;                       // tiles' scalars and masks: a tile's are read before the second tile after it is converted
constexpr float kOff = 7.f, kRaise = 8.f;

struct alignas(16) Meta {                      // read as 16-byte vectors
  float ks[4], vs_log2[4], vs_inv[4];          // per 32 tokens
  uint32_t k_apart[4], v_apart[4];             // scales are not in the codes, but only
  uint32_t valid[4];
  float col_ks[128], col_lv[128], col_rv[128]; // per token, for tiles that are not treated as a whole
};

template <int D> struct Lay {
  static constexpr int HALF = 128 * 128;                           // 128 rows of 64 channels, 128-byte rows, 128-byte swizzle
  static constexpr int TILE = HALF * (D / 64);
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, END = 6 * TILE;
  static constexpr int SMEM = END + 1024;                          // base rounded up to 1024
};

struct Shared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], q_full[2], o_full[2];
  uint64_t x_full, x_empty, drain;
  uint32_t tmem;
  int abort, never;                            // set by a wait that gave up; never set
  Meta meta[kMeta];
  float2 xml[128];
  KvPlaceScratch place;
};

// Descriptor of an MN-major operand: 64 channels per 128-byte row with 128-byte swizzle, 8-token groups 1024 bytes apart, blocks
// of 64 channels 16 KB apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// finite positive maximum -> the power of two at or above it (1 if there is none); at least 2^-80
__device__ __forceinline__ int pow2_above(uint32_t bits) {
  if (bits == 0) return 0;
  const int e = (int)(bits >> 23) - 127 + ((bits & 0x7fffffu) ? 1 : 0);
  return min(max(e, -80), 126);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Keys: the power of two that brings the largest code near the end of fp16's range, so that scales 2^12 apart still give normal
// fp16 numbers.  Values: none.  It would come out of the weights' range: P holds p VS, and tiles whose scales are not folded hold p vs,
// so with room for the values weights of 2^-9 of the largest were subnormal numbers already (4 bits, a tree's draft tile beside its
// cached ones).  Without it e4m3's subnormal codes allow scales 2^5 apart, whole numbers 2^12.
template <int FMT> constexpr int kRoom = FMT == GL_KV_FP8 ? 7 : FMT == GL_KV_INT8 ? 8 : 12;
constexpr int kSpread = 12;
template <int FMT> constexpr int kSpreadV = FMT == GL_KV_FP8 ? 5 : 12;

// scale ratio as two fp16 numbers (high, rest) of one value
__device__ __forceinline__ uint32_t split_half(float r) {
  const __half hi = __float2half_rn(r), lo = __float2half_rn(r - __half2float(hi));
  return (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
}
__device__ __forceinline__ uint32_t scaled(uint32_t x, uint32_t hi2, uint32_t lo2) {
  const __half2 v = *reinterpret_cast<__half2*>(&x), h = *reinterpret_cast<__half2*>(&hi2), l = *reinterpret_cast<__half2*>(&lo2);
  const __half2 r = __hfma2(v, h, __hmul2(v, l));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 32 lanes x 16 columns (x 8 for the store): for the paths that are kept small
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_8(uint32_t taddr, const uint32_t (&r)[8]) {      // tmem_st_wait() must follow
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {      // tmem_st_wait() must follow
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// a bounded wait of a whole warp: its lanes go on together, or give up together
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, nullptr, 0));
}

// ---- conversion warps ------------------------------------------------------------------------------------------------------
template <int D, int FMT> struct Conv {
  static constexpr int RB = FMT == GL_KV_INT4 ? D / 2 : D, CPT = RB / 16, N = 32 * RB / 16 / 32;    // N: 16-byte pieces per lane
  static constexpr int TPI = 32 / CPT;                                                              // tokens per instruction
  // token (of TPI) and 16-byte piece of its row that a lane takes: eight lanes that store together hold two tokens and, of
  // 128-byte rows, one half each, which the swizzle spreads over all banks
  static __device__ __forceinline__ int token(int lane) { return CPT == 8 ? (lane >> 4) * 2 + ((lane >> 2) & 1) : lane / CPT; }
  static __device__ __forceinline__ int piece(int lane) { return CPT == 8 ? ((lane >> 3) & 1) * 4 + (lane & 3) : lane % CPT; }

  // 16 bytes of token row `tok` -> fp16, times the token's ratio, into the swizzled tile
  static __device__ __forceinline__ void put(uint8_t* tile, int tok, int ch, const uint4& u, uint32_t ratio, uint32_t zero) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    const uint32_t hi = __byte_perm(ratio, 0, 0x1010), lo = __byte_perm(ratio, 0, 0x3232);
    constexpr int CH = FMT == GL_KV_INT4 ? 4 : 2;          // 16-byte chunks of fp16 that come out
    uint32_t o[CH * 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (FMT == GL_KV_INT4) {
        uint32_t n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] = kv_nibbles(w[i] >> (4 * j), zero);            // channels (j, j + 4)
        o[4 * i] = __byte_perm(n[0], n[1], 0x5410);
        o[4 * i + 1] = __byte_perm(n[2], n[3], 0x5410);
        o[4 * i + 2] = __byte_perm(n[0], n[1], 0x7632);
        o[4 * i + 3] = __byte_perm(n[2], n[3], 0x7632);
      } else {
        kv_bytes<FMT>(w[i], o[2 * i], o[2 * i + 1]);
      }
    }
    const int c0 = ch * CH;
    uint8_t* row = tile + (c0 >> 3) * Lay<D>::HALF + tok * 128;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      *reinterpret_cast<uint4*>(row + ((((c0 & 7) + i) ^ (tok & 7)) << 4)) =
          make_uint4(scaled(o[4 * i], hi, lo), scaled(o[4 * i + 1], hi, lo), scaled(o[4 * i + 2], hi, lo), scaled(o[4 * i + 3], hi, lo));
  }
};

// One code for keys and values (`values`): the four roles' inner loops together have to stay in the instruction caches, and
// are kept small for it.  Of every tile the warp takes the tokens 32 w .. 32 w + 31 (lane = token where scales are meant).
template <int D, int FMT>
__device__ __forceinline__ void convert_role(const KvAttendParams& p, Shared& sh, uint8_t* base, KvWalk<kKvTcRows> walk, const bool values) {
  using C = Conv<D, FMT>;
  constexpr int G = C::N < 4 ? C::N : 4;                                  // pieces in registers; a tile is N / G groups of them
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) & 3, c_tok = C::token(lane), c_piece = C::piece(lane);
  volatile int* abort = &sh.abort;
  const KvBatch& kb = p.kb;
  const uint8_t* codes = (values ? p.v_codes : p.k_codes) + c_piece * 16;
  const float* scales = values ? p.v_scales : p.k_scales;
  const uint8_t* zeros = values ? p.v_zeros : p.k_zeros;
  uint64_t* full_bar = values ? sh.v_full : sh.k_full;
  uint64_t* empty_bar = values ? sh.v_empty : sh.k_empty;
  uint8_t* tiles = base + (values ? Lay<D>::V : Lay<D>::K);

  KvPiece pc;
  bool have;
  int tile, parted;                                                       // parted: first tile that not every row of the unit sees all of
  auto next_piece = [&]() {
    have = walk.next(p, blockIdx.x, pc);
    tile = have ? pc.t0 : 0;
    parted = have ? (pc.s.ctx + (p.mask == nullptr ? pc.row0 / p.group + 1 : 0)) / kKvTile : 0;
  };
  next_piece();
  // A tile two ahead: its page numbers are on their way while the codes of the one before are fetched.
  struct Item { int page, place, head; uint32_t flags; };                 // flags: 1 tile exists, 2 token within the sequence, 4 parted
  auto fetch = [&]() {
    Item it{-1, 0, 0, 0u};
    while (have && tile >= pc.t1) next_piece();
    if (have) {
      const int pos = tile * kKvTile + w * 32 + lane;
      it.head = pc.head;
      it.flags = 1u | (tile >= parted ? 4u : 0u);
      if (pos < pc.s.len) {
        const int pi = p.page_shift >= 0 ? pos >> p.page_shift : pos / kb.page_size;
        it.place = pos - pi * kb.page_size;
        it.page = kv_load(kb.page_table + (int64_t)walk.b * kb.pt_stride + pi);
        it.flags |= 2u;
      }
      ++tile;
    }
    return it;
  };
  auto slot_of = [&](const Item& it) -> uint32_t { return it.flags & 2u ? kv_slot32(kb, it.page, it.head, it.place) : kNoSlot; };
  // rows that follow each other (32 tokens inside one page) need one address, others one each
  struct Rows { uint32_t slot; bool in_line; const uint8_t* at; };
  auto rows_of = [&](const Item& it) {
    Rows r;
    r.slot = slot_of(it);
    const uint32_t s0 = __shfl_sync(0xffffffffu, r.slot, 0);
    r.in_line = __all_sync(0xffffffffu, r.slot != kNoSlot && r.slot == s0 + lane);
    r.at = codes + ((int64_t)s0 + c_tok) * C::RB;
    return r;
  };
  auto take = [&](const Rows& r, int piece) {
    if (r.in_line) return kv_load(reinterpret_cast<const uint4*>(r.at + piece * (C::TPI * C::RB)));
    const uint32_t s = __shfl_sync(0xffffffffu, r.slot, c_tok + piece * C::TPI);
    return s != kNoSlot ? kv_load(reinterpret_cast<const uint4*>(codes + (int64_t)s * C::RB)) : make_uint4(0, 0, 0, 0);
  };

  Item nxt = fetch();
  if (!(nxt.flags & 1u)) return;
  Rows rows = rows_of(nxt);
  uint32_t flags = nxt.flags;
  nxt = fetch();
  uint4 u[G];
#pragma unroll
  for (int i = 0; i < G; ++i) u[i] = take(rows, i);
  float scale = rows.slot != kNoSlot ? kv_load(scales + rows.slot) : 0.f;
  uint32_t zero = FMT == GL_KV_INT4 && rows.slot != kNoSlot ? kv_load(zeros + rows.slot) : 0u;

#pragma unroll 1
  for (int n = 0; flags & 1u; ++n) {
    const int st = n & 1;
    const bool in_part = flags & 4u;
    // the power of two, and whether the scales are near enough to each other
    const uint32_t bits = __float_as_uint(scale);
    const bool plain = bits - 1u < 0x7f7fffffu;                          // positive and finite
    const uint32_t hi = __reduce_max_sync(0xffffffffu, plain ? bits : 0u), lo = __reduce_min_sync(0xffffffffu, plain ? bits : 0x7f7fffffu);
    const bool apart = in_part || (int)(hi >> 23) - (int)(lo >> 23) >= (values ? kSpreadV<FMT> : kSpread);
    const int e = apart ? 0 : pow2_above(hi) - (values ? 0 : kRoom<FMT>);
    const bool number = fabsf(scale) < INFINITY, none = apart && scale < kTinyScale;
    const uint32_t valid = __ballot_sync(0xffffffffu, rows.slot != kNoSlot);
    // Values that are not numbers would reach every row through P V', so V' is 0 there, and the exponent is NaN, which only the
    // rows that see the token meet.  (e4m3's NaN codes matter where some rows do not see the token.)
    uint32_t bad = values ? __ballot_sync(0xffffffffu, !number) : 0u;
    const uint32_t ratio = !number ? (values ? 0u : 0x00007fffu) : values && none ? 0u : apart ? 0x00003c00u : split_half(scale * pow2(-e));
    const uint32_t zz = (0x6400u + zero) * 0x10001u;
    const Rows rows_next = rows_of(nxt);

    if (n >= 2 && !warp_wait(&empty_bar[st], ((n >> 1) & 1) ^ 1, abort)) return;
    uint8_t* dst = tiles + st * Lay<D>::TILE;
#pragma unroll 1
    for (int g = 0; g < C::N; g += G) {
      const bool last = g + G >= C::N;                                    // then the pieces of the next tile follow
      Rows from;
      from.slot = last ? rows_next.slot : rows.slot;
      from.in_line = last ? rows_next.in_line : rows.in_line;
      from.at = last ? rows_next.at : rows.at;
      const int base_piece = last ? 0 : g + G;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int t = c_tok + (g + i) * C::TPI;
        if (FMT == GL_KV_FP8 && values && in_part) {
          const uint32_t m = 0x7f7f7f7fu, one = 0x01010101u;
          const bool nan = (((((u[i].x & m) + one) | ((u[i].y & m) + one) | ((u[i].z & m) + one) | ((u[i].w & m) + one)) & 0x80808080u) != 0);
          const uint32_t who = __reduce_or_sync(0xffffffffu, nan ? 1u << t : 0u);
          if ((who >> t) & 1u) u[i] = make_uint4(0, 0, 0, 0);
          bad |= who;
        }
        const uint32_t r = __shfl_sync(0xffffffffu, ratio, t), z = FMT == GL_KV_INT4 ? __shfl_sync(0xffffffffu, zz, t) : 0u;
        C::put(dst, w * 32 + t, c_piece, u[i], r, z);
        u[i] = take(from, base_piece + i);
      }
    }
    Meta& m = sh.meta[n % kMeta];
    if (lane == 0) {
      if (values) {
        m.vs_log2[w] = (float)e;
        m.vs_inv[w] = pow2(-e);
        m.v_apart[w] = apart || bad;
      } else {
        m.ks[w] = pow2(e);
        m.k_apart[w] = apart;
        m.valid[w] = valid;
      }
    }
    if (values) {
      const float v = none ? kTinyScale : scale;
      m.col_lv[w * 32 + lane] = (bad >> lane) & 1u ? __int_as_float(0x7fc00000) : apart ? __log2f(v) : (float)e;
      m.col_rv[w * 32 + lane] = apart ? __frcp_rn(v) : pow2(-e);
    } else {
      m.col_ks[w * 32 + lane] = apart ? scale : pow2(e);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full_bar[st]);
    flags = nxt.flags;
    rows = rows_next;
    if (flags & 1u) {
      scale = rows.slot != kNoSlot ? kv_load(scales + rows.slot) : 0.f;
      if (FMT == GL_KV_INT4) zero = rows.slot != kNoSlot ? kv_load(zeros + rows.slot) : 0u;
      nxt = fetch();
    }
  }
}

// ---- the MMA lane ------------------------------------------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void mma_role(const KvAttendParams& p, Shared& sh, uint32_t base, KvWalk<kKvTcRows> walk, uint32_t idesc_s, uint32_t idesc_o) {
  volatile int* abort = &sh.abort;
  const uint32_t tm = sh.tmem;
  // descriptors as halves: the high words are constant, the low words step with the address
  const uint64_t qd = smem_desc_sw128(base + Lay<D>::Q), kd = smem_desc_sw128(base + Lay<D>::K), vd = desc_mn(base + Lay<D>::V);
  const uint32_t q_lo = (uint32_t)qd, k_lo = (uint32_t)kd, k_hi = (uint32_t)(kd >> 32), v_lo = (uint32_t)vd, v_hi = (uint32_t)(vd >> 32);
  KvPiece pc;
  int n0 = 0;                                  // tiles of earlier pieces
  uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
  while (walk.next(p, blockIdx.x, pc)) {
    const int n = pc.t1 - pc.t0;
    if (n <= 0) continue;
    const bool both = pc.rows > 128;
    const int events = both ? 2 * n : n;
    auto scores = [&](int e) -> bool {
      const int s = e & 1, j = n0 + (both ? e >> 1 : e), st = j & 1;
      if ((!both || s == 0) && !mbar_wait_spin(&sh.k_full[st], (j >> 1) & 1, abort, nullptr, 0)) return false;
      tc_fence_after();
      const uint32_t q = q_lo + s * (Lay<D>::TILE >> 4), k = k_lo + st * (Lay<D>::TILE >> 4);
#pragma unroll 1
      for (int half = 0; half < D / 64; ++half)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss_f16_lohi(tm + s * 128, q + half * (Lay<D>::HALF >> 4) + kk * 2, k + half * (Lay<D>::HALF >> 4) + kk * 2, k_hi, idesc_s, half + kk > 0);
      tc_commit(&sh.s_full[s]);
      if (!both || s == 1) tc_commit(&sh.k_empty[st]);
      return true;
    };
    for (int s = 0; s < 2 && s < events; ++s) {                          // (a stream without a tile loads no queries)
      if (!mbar_wait_spin(&sh.q_full[s], q_phase[s], abort, nullptr, 0)) return;
      q_phase[s] ^= 1;
    }
    tc_fence_after();
    for (int e = 0; e < 2 && e < events; ++e)
      if (!scores(e)) return;
    for (int e = 0; e < events; ++e) {
      const int s = e & 1, i = both ? e >> 1 : e, j = n0 + i, st = j & 1;
      if ((!both || s == 0) && !mbar_wait_spin(&sh.v_full[st], (j >> 1) & 1, abort, nullptr, 0)) return;
      if (!mbar_wait_spin(&sh.p_full[s], p_phase[s], abort, nullptr, 0)) return;
      p_phase[s] ^= 1;
      tc_fence_after();
      const uint32_t v = v_lo + st * (Lay<D>::TILE >> 4);
#pragma unroll 1
      for (int k2 = 0; k2 < 8; k2 += 4)
#pragma unroll
        for (int kk = k2; kk < k2 + 4; ++kk)
          mma_ts_f16_lohi(tm + 256 + s * D, tm + s * 128 + kk * 8, v + kk * 128, v_hi, idesc_o, e >= 2 || kk > 0);
      if (!both || s == 1) tc_commit(&sh.v_empty[st]);
      if (e + 2 >= events) tc_commit(&sh.o_full[s]);
      else if (!scores(e + 2)) return;
    }
    n0 += n;
  }
}

// ---- the two streams ---------------------------------------------------------------------------------------------------------
template <int D, typename T>
__device__ __forceinline__ void stream_role(const KvAttendParams& p, Shared& sh, uint8_t* base, KvWalk<kKvTcRows> walk) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, s = warp >> 2, row = threadIdx.x & 127;
  volatile int* abort = &sh.abort;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t ts = sh.tmem + lanes + s * 128, to = sh.tmem + lanes + 256 + s * D;
  KvPiece pc;
  int n0 = 0, merges = 0;
  uint32_t s_phase = 0, o_phase = 0;
  bool ok = true;
  KvCut cut{};
  while (walk.next(p, blockIdx.x, pc)) {
    KvWalk<kKvTcRows>::note(cut, pc);
    const int n = pc.t1 - pc.t0 > 0 ? pc.t1 - pc.t0 : 0;
    const bool both = pc.rows > 128;
    const int r = both ? s * 128 + row : row;                    // row of the unit
    const bool live = r < pc.rows;
    const int rr = pc.row0 + (live ? r : 0), tok = rr / p.group, head = pc.head * p.group + (rr - tok * p.group);
    const bool any_live = __any_sync(0xffffffffu, live);
    float m_used = -INFINITY, l = 0.f;
    const int mine = both ? n : s == 0 ? (n + 1) / 2 : n / 2;
    if (mine > 0 && ok) {
      // ---- queries: fp16 by a power of two, into this stream's swizzled tile
      if (merges > 0) ok = warp_wait(&sh.x_empty, (merges - 1) & 1, abort);
      const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(pc.s.first + tok) * p.q_sn + (int64_t)head * p.q_sh;
      float factor = 1.f, inv = 1.f;
      if constexpr (!IsHalf<T>::value) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint4 u = live ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
        }
        const int ex = min(max((int)(top >> 7), 1), 253);
        inv = __int_as_float((254 - ex) << 23);
        factor = __int_as_float(ex << 23);
      }
      // the sign of the scale goes into the queries: maxima are taken of the scores themselves
      const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
      const float qs = fabsf(p.scale_log2) * factor;
      uint8_t* qt = base + Lay<D>::Q + s * Lay<D>::TILE + row * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        uint4 u = live ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (!IsHalf<T>::value) {
            const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * inv, __uint_as_float(w[j] & 0xffff0000u) * inv);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          w[j] ^= flip;
        }
        *reinterpret_cast<uint4*>(qt + (i >> 3) * Lay<D>::HALF + (((i & 7) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full[s]);

      const int t_lo = (pc.row0 + (both ? s * 128 : 0)) / p.group;      // the stream's first row's token
      for (int i = 0; i < mine && ok; ++i) {
        const int j = both ? i : 2 * i + s;
        const Meta& meta = sh.meta[(n0 + j) % kMeta];
        ok = warp_wait(&sh.s_full[s], s_phase, abort) && warp_wait(&sh.v_full[(n0 + j) & 1], ((n0 + j) >> 1) & 1, abort);     // (the values' scales)
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after();
        if (!any_live) {                                              // 32 rows of nobody: their weights may be anything
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[s]);
          continue;
        }
        const int tile0 = (pc.t0 + j) * kKvTile;
        const uint4 vld = *reinterpret_cast<const uint4*>(meta.valid), ka = *reinterpret_cast<const uint4*>(meta.k_apart), va = *reinterpret_cast<const uint4*>(meta.v_apart);
        const bool full = (ka.x | ka.y | ka.z | ka.w | va.x | va.y | va.z | va.w) == 0 && (vld.x & vld.y & vld.z & vld.w) == 0xffffffffu &&
                          tile0 + kKvTile <= pc.s.ctx + (p.mask == nullptr ? t_lo + 1 : 0);
        uint32_t seen[4] = {vld.x, vld.y, vld.z, vld.w};
        if (!full) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int at = tile0 + 32 * w - pc.s.ctx;                  // the word's first token: which new token
            if (at + 32 <= 0) continue;
            if (p.mask == nullptr) {
              const int k = tok + 1 - at;
              seen[w] &= k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u;
            } else {
              const uint8_t* mk = p.mask + (int64_t)(pc.s.first + tok) * p.mask_stride;
              for (int k = max(0, -at); k < 32; ++k)
                if ((seen[w] >> k) & 1u)
                  if (at + k >= p.mask_cols || mk[at + k] == 0) seen[w] &= ~(1u << k);
            }
          }
        }
        // ---- the tile's maximum.  (The paths for tiles that are not full are rolled up: unrolled, the kernel outgrew the
        // instruction cache and ran at less than half its speed.)
        // columns c .. c + 15 that this row sees; whether any token of theirs exists
        auto seen16 = [&](int c) { return ((c < 64 ? (c < 32 ? seen[0] : seen[1]) : (c < 96 ? seen[2] : seen[3])) >> (c & 31)) & 0xffffu; };
        auto there16 = [&](int c) { return (meta.valid[c >> 5] >> (c & 31)) & 0xffffu; };
        float t_top = -INFINITY;
        if (full) {
          uint32_t x[32];
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            tmem_ld_32x32(ts + 32 * h, x);
            tmem_ld_fence(x);
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 32; k += 2) top = max3(top, __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
            t_top = fmaxf(t_top, fmaf(top, qs * meta.ks[h], meta.vs_log2[h]));
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            if (there16(c) == 0) continue;
            uint32_t y[16];
            tmem_ld_16(ts + c, y);
            const uint32_t sw = seen16(c);
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const float4 ks = *reinterpret_cast<const float4*>(meta.col_ks + c + k), lv = *reinterpret_cast<const float4*>(meta.col_lv + c + k);
              const float t0 = fmaf(__uint_as_float(y[k]) * ks.x, qs, lv.x), t1 = fmaf(__uint_as_float(y[k + 1]) * ks.y, qs, lv.y);
              const float t2 = fmaf(__uint_as_float(y[k + 2]) * ks.z, qs, lv.z), t3 = fmaf(__uint_as_float(y[k + 3]) * ks.w, qs, lv.w);
              t_top = fmaxf(t_top, fmaxf(fmaxf((sw >> k) & 1u ? t0 : -INFINITY, (sw >> (k + 1)) & 1u ? t1 : -INFINITY),
                                         fmaxf((sw >> (k + 2)) & 1u ? t2 : -INFINITY, (sw >> (k + 3)) & 1u ? t3 : -INFINITY)));
            }
          }
        }
        const bool raise = t_top > m_used + kRaise || (m_used == -INFINITY && t_top != -INFINITY);
        if (__any_sync(0xffffffffu, raise)) {
          const float m_new = raise ? t_top : m_used, f = raise ? kv_exp2(m_used - m_new) : 1.f;
          l *= f;
          m_used = m_new;
          if (i > 0) {                                                // (s_full: the products before this tile's scores are done)
            uint32_t x[1][32];
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              tmem_ld_32x32(to + d, x[0]);
              tmem_ld_fence(x[0]);
#pragma unroll
              for (int k = 0; k < 32; ++k) x[0][k] = __float_as_uint(__uint_as_float(x[0][k]) * f);
              tmem_st_32x32(to + d, x[0]);
            }
          }
        }
        // ---- weights, over the scores
        const float to_p = m_used == -INFINITY ? 0.f : kOff - m_used;
        if (full) {
          uint32_t x[32];
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            tmem_ld_32x32(ts + 32 * h, x);
            tmem_ld_fence(x);
            const float a = qs * meta.ks[h], sub = meta.vs_log2[h] + to_p;
            const uint64_t a2 = pack2(a, a), sub2 = pack2(sub, sub);
            uint64_t sum2 = 0ull;
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float e0, e1;
              unpack2(fma2(pack2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), a2, sub2), e0, e1);
              e0 = kv_exp2(e0);
              e1 = kv_exp2(e1);
              sum2 = add2(sum2, pack2(e0, e1));
              const __half2 hh = __floats2half2_rn(e0, e1);
              pk[k >> 1] = *reinterpret_cast<const uint32_t*>(&hh);
            }
            float s0, s1;
            unpack2(sum2, s0, s1);
            l = fmaf(s0 + s1, meta.vs_inv[h], l);
            tmem_st_16(ts + h * 16, pk);                              // (columns whose scores have been read)
          }
          tmem_st_wait();
        } else {
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            uint32_t pk[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (there16(c) != 0) {
              uint32_t y[16];
              tmem_ld_16(ts + c, y);
              const uint32_t sw = seen16(c);
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                const float4 ks = *reinterpret_cast<const float4*>(meta.col_ks + c + k), lv = *reinterpret_cast<const float4*>(meta.col_lv + c + k),
                             rv = *reinterpret_cast<const float4*>(meta.col_rv + c + k);
                // (a token that is not seen has the weight 0, whatever its scale)
                const float e0 = (sw >> k) & 1u ? kv_exp2(fmaf(__uint_as_float(y[k]) * ks.x, qs, lv.x) + to_p) : 0.f;
                const float e1 = (sw >> (k + 1)) & 1u ? kv_exp2(fmaf(__uint_as_float(y[k + 1]) * ks.y, qs, lv.y) + to_p) : 0.f;
                const float e2 = (sw >> (k + 2)) & 1u ? kv_exp2(fmaf(__uint_as_float(y[k + 2]) * ks.z, qs, lv.z) + to_p) : 0.f;
                const float e3 = (sw >> (k + 3)) & 1u ? kv_exp2(fmaf(__uint_as_float(y[k + 3]) * ks.w, qs, lv.w) + to_p) : 0.f;
                l += ((sw >> k) & 1u ? e0 * rv.x : 0.f) + ((sw >> (k + 1)) & 1u ? e1 * rv.y : 0.f) + ((sw >> (k + 2)) & 1u ? e2 * rv.z : 0.f) + ((sw >> (k + 3)) & 1u ? e3 * rv.w : 0.f);
                pk[k >> 1] = kv_pair<__half>(e0, e1);
                pk[(k >> 1) + 1] = kv_pair<__half>(e2, e3);
              }
            }
            tmem_st_8(ts + c / 2, pk);                                // (columns whose scores have been read)
            tmem_st_wait();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[s]);
      }
      if (ok) {
        ok = warp_wait(&sh.o_full[s], o_phase, abort);
        o_phase ^= 1;
        tc_fence_after();
      }
    }

    // ---- the result of the unit, or of its part
    const bool merge = !both && n > 1;
    float m1 = -INFINITY, l1 = 0.f;
    const float4* other = reinterpret_cast<const float4*>(base + Lay<D>::Q) + row;      // [D / 4][128]: the streams' queries are done with
    if (merge && s == 1) {
      uint32_t x[32];
      if (ok) {
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          tmem_ld_32x32(to + d, x);
          tmem_ld_fence(x);
#pragma unroll
          for (int k = 0; k < 8; ++k) const_cast<float4*>(other)[(d / 4 + k) * 128] = make_float4(__uint_as_float(x[4 * k]), __uint_as_float(x[4 * k + 1]), __uint_as_float(x[4 * k + 2]), __uint_as_float(x[4 * k + 3]));
        }
        sh.xml[row] = make_float2(m_used, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.x_full);
      }
    }
    if (both || s == 0) {
      if (merge && ok) {
        ok = warp_wait(&sh.x_full, merges & 1, abort);
        const float2 ml = sh.xml[row];
        m1 = ml.x;
        l1 = ml.y;
      }
      const float top = fmaxf(m_used, m1);
      const float f0 = m_used == -INFINITY ? (l == 0.f ? 0.f : 1.f) : kv_exp2(m_used - top), f1 = m1 == -INFINITY ? (l1 == 0.f ? 0.f : 1.f) : kv_exp2(m1 - top);
      float lt = l * f0 + l1 * f1;
      if (!ok) lt = __int_as_float(0x7fc00000);                     // a wait ran out: the rows say so
      const float rcp = lt == 0.f ? 0.f : 1.f / lt;
      uint32_t x[32];
      T* dst = reinterpret_cast<T*>(p.out) + ((int64_t)(pc.s.first + tok) * p.hq + head) * D;
      const int64_t pr = (int64_t)pc.slot * kKvTcRows + r;
#pragma unroll 1
      for (int d = 0; d < D; d += 32) {
        if (mine > 0) {
          tmem_ld_32x32(to + d, x);
          tmem_ld_fence(x);
        }
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = mine > 0 ? __uint_as_float(x[k]) * f0 : 0.f;
        if (merge) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 y = other[(d / 4 + k) * 128];
            v[4 * k] = fmaf(y.x, f1, v[4 * k]);
            v[4 * k + 1] = fmaf(y.y, f1, v[4 * k + 1]);
            v[4 * k + 2] = fmaf(y.z, f1, v[4 * k + 2]);
            v[4 * k + 3] = fmaf(y.w, f1, v[4 * k + 3]);
          }
        }
        if (live) {
          if (pc.whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float a0 = lt == 0.f ? 0.f : v[8 * k + 2 * j] * rcp, a1 = lt == 0.f ? 0.f : v[8 * k + 2 * j + 1] * rcp;
                if constexpr (IsHalf<T>::value) {
                  const __half2 h = __floats2half2_rn(a0, a1);
                  o[j] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                  const __nv_bfloat162 h = __floats2bfloat162_rn(a0, a1);
                  o[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
              }
              *reinterpret_cast<uint4*>(dst + d + 8 * k) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) *reinterpret_cast<float4*>(p.part_o + pr * D + d + 4 * k) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          }
        }
      }
      if (live && !pc.whole) p.part_ml[pr] = make_float2(top, lt);
      tc_fence_before();
      if (merge && s == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.x_empty);
      }
    }
    if (merge) ++merges;
    n0 += n;
  }
  if (threadIdx.x == 0 && p.cuts != nullptr) p.cuts[blockIdx.x] = cut;
}

template <int D, int FMT, typename T>
__global__ void __launch_bounds__(kThreads, 1) kv_attend_tc_kernel(const KvAttendParams p, uint32_t idesc_s, uint32_t idesc_o) {
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  uint8_t* base = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], 4);
      mbar_init(&sh.v_full[i], 4);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.q_full[i], 4);
      mbar_init(&sh.o_full[i], 1);
    }
    mbar_init(&sh.x_full, 4);
    mbar_init(&sh.x_empty, 4);
    mbar_init(&sh.drain, 1);
    sh.abort = sh.never = 0;
    fence_barrier_init();
  }
  if (warp == 16) tmem_alloc(&sh.tmem, 512);
  gl_launch_dependents();
  gl_grid_dependency_wait();
  KvWalk<kKvTcRows> walk;
  walk.start(p, kv_place_of_block<kKvTcRows, kThreads>(p, blockIdx.x, sh.place), blockIdx.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  // Every wait is bounded; one that gives up ends all roles, the rows that it leaves unfinished become NaN, and the status says so.
  // Registers: 640 threads are launched with 96 each; 2 x 128 + 2 x 88 + 48 = 480 = 5 x 96 are shared out again.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    stream_role<D, T>(p, sh, base, walk);
  } else if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    convert_role<D, FMT>(p, sh, base, walk, warp >= 12);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (threadIdx.x == 16 * 32) {
      mma_role<D>(p, sh, smem_u32(base), walk, idesc_s, idesc_o);
      // nothing of this block's is in flight when the TMEM goes back
      tc_commit(&sh.drain);
      mbar_wait(&sh.drain, 0, &sh.never, nullptr, 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && (sh.abort | sh.never) != 0) atomicOr(&g_wait_status, sh.abort | sh.never << 1);
  if (warp == 16) tmem_dealloc(sh.tmem, 512);
}

template <int D, int FMT, typename T>
int launch(const KvAttendParams& p, cudaStream_t st) {
  if (int rc = kv_allow_smem((const void*)kv_attend_tc_kernel<D, FMT, T>, Lay<D>::SMEM)) return rc;
  const uint32_t idesc_s = gl_idesc(1, 0, 0, 128, kKvTile), idesc_o = gl_idesc(1, 0, 0, 128, D) | (1u << 16);     // bit 16: B is MN-major
  GL_CUDA_CHECK(gl_launch_pdl(kv_attend_tc_kernel<D, FMT, T>, dim3((unsigned)p.blocks), dim3(kThreads), Lay<D>::SMEM, st, p, idesc_s, idesc_o));
  return GL_OK;
}
template <int D, typename T>
int launch_fmt(const KvAttendParams& p, int fmt, cudaStream_t st) {
  switch (fmt) {
    case GL_KV_FP8: return launch<D, GL_KV_FP8, T>(p, st);
    case GL_KV_INT8: return launch<D, GL_KV_INT8, T>(p, st);
    default: return launch<D, GL_KV_INT4, T>(p, st);
  }
}

}  // namespace

extern "C" int gl_kv_attend_status(int32_t* status, int32_t clear, void* stream) {
  if (status == nullptr) GL_FAIL(GL_E_INVALID, "gl_kv_attend_status: null argument");
  cudaStream_t st = (cudaStream_t)stream;
  int now = 0;
  GL_CUDA_CHECK(cudaMemcpyFromSymbolAsync(&now, g_wait_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  GL_CUDA_CHECK(cudaStreamSynchronize(st));
  *status = now;
  if (now != 0 && clear) {
    now = 0;
    GL_CUDA_CHECK(cudaMemcpyToSymbolAsync(g_wait_status, &now, sizeof(int), 0, cudaMemcpyHostToDevice, st));
    GL_CUDA_CHECK(cudaStreamSynchronize(st));
  }
  return GL_OK;
}

int gl_kv_attend_tc_launch(const KvAttendParams& p, int head_dim, int format, int x_dtype, cudaStream_t st) {
  if (head_dim == 128) return x_dtype == GL_BF16 ? launch_fmt<128, __nv_bfloat16>(p, format, st) : launch_fmt<128, __half>(p, format, st);
  return x_dtype == GL_BF16 ? launch_fmt<64, __nv_bfloat16>(p, format, st) : launch_fmt<64, __half>(p, format, st);
}
