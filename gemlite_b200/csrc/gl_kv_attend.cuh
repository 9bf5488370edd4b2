// What the two attention kernels over the quantised cache share: parameters, exact conversion of codes to fp16, output.
#pragma once
#include "gl_kv.cuh"

// what a block says about the units that its borders cut: bit 0: its last piece begins a unit and does not finish it (the unit:
// first row of the sequence's tokens, head, first row, rows); bit 1: its first piece goes on with a unit; bit 2: and finishes it
struct alignas(16) KvCut {
  int32_t flags, first, head, row0, rows, pad[3];
};
struct KvAttendParams {
  KvBatch kb;
  const uint8_t *k_codes, *v_codes, *k_zeros, *v_zeros;
  const float *k_scales, *v_scales;
  const void* q;
  void* out;
  const uint8_t* mask;
  float* part_o;               // [2 * blocks][rows of a unit][D], unnormalised
  float2* part_ml;             // [2 * blocks][rows of a unit]: maximum and sum (0: nothing seen)
  KvCut* cuts;                 // [blocks]
  int64_t q_sn, q_sh, mask_stride;
  int32_t mask_cols, hq, group, page_shift, blocks;
  float scale_log2;
};

// the tcgen05 kernel (gl_kv_attend_tc.cu): 256 query rows of a kv head per unit, one block per SM
constexpr int kKvTcRows = 256;
// opt-in to more than 48 KB of dynamic shared memory on the current device, once per kernel
int kv_allow_smem(const void* kernel, int bytes);
int gl_kv_attend_tc_launch(const KvAttendParams& p, int head_dim, int format, int x_dtype, cudaStream_t st);

// Values whose scale is smaller count as zero: their codes become zeros under this scale.  Their term of the denominator is at most
// 2^15 / kTinyScale, 2^95, so that the 2^30 tokens that a table may hold stay below 2^126.  (With 1e-30, 2^115, a
// dozen thousand slots that were never written made it infinite, and the row zero.)
constexpr float kTinyScale = 1e-24f;

template <typename T> struct IsHalf { static constexpr bool value = false; };
template <> struct IsHalf<__half> { static constexpr bool value = true; };

#ifdef __CUDACC__
// Page numbers, codes and scales: from L2.  Not by the read-only path (ld.global.nc), which is for memory that nobody writes
// during a kernel: this launch may begin while the write that it waits for still runs.  (Codes by L1: a chunk of 1000 tokens over 7000
// 408 us, past it 402.)
template <typename V> __device__ __forceinline__ V kv_load(const V* p) { return __ldcg(p); }

// row of a token's (page, head, place) in the cache as a 32-bit number (gl_kv_check: there are fewer than 2^32 - 1)
constexpr uint32_t kNoSlot = 0xffffffffu;
__device__ __forceinline__ uint32_t kv_slot32(const KvBatch& kb, int page, int head, int place) {
  return (unsigned)page < (unsigned)kb.num_pages ? ((uint32_t)page * (uint32_t)kb.hkv + (uint32_t)head) * (uint32_t)kb.page_size + (uint32_t)place : kNoSlot;
}

// ---- how the work is dealt out
// A unit is ROWS query rows (token, head of the group) of one kv head of one sequence; it is worked through in tiles of kKvTile cached
// tokens.  All units' tiles stand in one line (sequence, kv head, row block, tile), and block i of n takes the i-th of n
// equal pieces of the line: lengths may differ as they like, every block gets the same number of tiles, and a unit is cut
// only where a block ends.  A block whose piece holds a whole unit writes the unit's result; the part of a unit that it starts in
// the middle of goes to its scratch slot 2 i, the part that it does not finish to slot 2 i + 1, and kv_attend_join_kernel joins
// them by what the blocks say in `cuts`.
// Nobody waits for anybody.  The lengths are on the device, so every block adds them up for itself.
constexpr int kKvTile = 128;

// Starting and finishing a unit (queries, scratch or output, the pipeline's ends) costs as much as some tiles: they stand before
// its tiles in the line, so that a block that gets many short units gets fewer tiles.  (Measured: 2 for units of 8 or 16 rows,
// 106 us against 113 with 1 on 32 decoding sequences of 500 to 16000 tokens; 4 for units of 256, 329 us against 341 with 2 on 8
// trees of 64.  The shortest calls pay for it: one token over 1000 cached took 9.6 us before there was a cost, 11.3 with it, because
// the grid is sized by tiles alone and blocks that get only cost do nothing.)
template <int ROWS> constexpr int kUnitCost = ROWS >= 256 ? 4 : 2;
struct KvSeq {
  int first, new_b, ctx, len, tiles, blocks;      // blocks: row blocks per kv head (0: no new tokens); tiles: with the cost
};
template <int ROWS> __device__ __forceinline__ KvSeq kv_seq(const KvAttendParams& p, int b) {
  KvSeq s;
  int end;
  kv_new_rows(p.kb, b, s.first, end);
  s.new_b = end - s.first;
  s.ctx = kv_len(p.kb, b);
  s.len = (int)min((int64_t)s.ctx + s.new_b, kv_capacity(p.kb));
  s.tiles = kUnitCost<ROWS> + max(1, (s.len + kKvTile - 1) / kKvTile);
  s.blocks = (int)(((int64_t)s.new_b * p.group + ROWS - 1) / ROWS);
  return s;
}
__device__ __forceinline__ int64_t kv_seq_work(const KvAttendParams& p, const KvSeq& s) { return (int64_t)p.kb.hkv * s.blocks * s.tiles; }

// 64-bit quotients of numbers that almost always have 32 (the general routine is a hundred instructions)
__device__ __forceinline__ int64_t kv_div(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// the line's pieces: the first `more` blocks get `each` + 1 tiles, the others `each`
struct KvShare {
  int64_t total, each;
  int more;
  __device__ __forceinline__ KvShare(int64_t t, int blocks) : total(t), each(kv_div(t, blocks)), more((int)(t - each * blocks)) {}
  __device__ __forceinline__ int64_t begin(int i) const { return each * i + min(i, more); }
};
// place in the line: sequence, and tiles of the sequence before it
struct KvPlace {
  int64_t total, prefix, off;      // tiles in all; tiles before the sequence; within it
  int b;                           // -1: behind the end
};
struct KvPlaceScratch {
  int64_t warp_sum[32];
  int64_t prefix, off;
  int b;
};
// Where block `i` of p.blocks begins (i = p.blocks: the end).  All THREADS threads of the block; ends with __syncthreads.
template <int ROWS, int THREADS> __device__ __forceinline__ KvPlace kv_place_of_block(const KvAttendParams& p, int i, KvPlaceScratch& sc) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = p.kb.batch;
  const int per = (B + THREADS - 1) / THREADS, lo = min(tid * per, B), hi = min(lo + per, B);
  int64_t sum = 0;
  for (int b = lo; b < hi; ++b) sum += kv_seq_work(p, kv_seq<ROWS>(p, b));
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sc.warp_sum[warp] = incl;
  if (tid == 0) sc.b = -1;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += sc.warp_sum[w];
    total += sc.warp_sum[w];
  }
  int64_t prefix = before + incl - sum;
  const int64_t x = KvShare(total, p.blocks).begin(i);
  if (x >= prefix && x < prefix + sum) {
    for (int b = lo; b < hi; ++b) {
      const int64_t w = kv_seq_work(p, kv_seq<ROWS>(p, b));
      if (x < prefix + w) {
        sc.b = b;
        sc.prefix = prefix;
        sc.off = x - prefix;
        break;
      }
      prefix += w;
    }
  }
  __syncthreads();
  KvPlace pl;
  pl.total = total;
  pl.b = sc.b;
  pl.prefix = sc.prefix;
  pl.off = sc.off;
  return pl;
}
// row blocks are taken from both ends in turn: without a mask, late ones see more tokens than early ones
__device__ __forceinline__ int kv_row_block(int i, int n) { return (i & 1) ? n - 1 - (i >> 1) : i >> 1; }

struct KvPiece {
  KvSeq s;
  int head, row0, rows;            // kv head; first row of the unit and its live rows
  int t0, t1;                      // tiles of this piece that some row may see (t1 <= t0: none)
  bool whole;                      // the unit's tiles are all in this piece
  bool ends;                       // its last ones are
  int slot;                        // else: scratch slot of its part
};
// walks a block's piece of the line, unit by unit
template <int ROWS> struct KvWalk {
  int b, left_valid;
  int64_t off, left;               // place within sequence b; tiles left to take
  bool at_start;
  KvSeq s;
  __device__ __forceinline__ void start(const KvAttendParams& p, const KvPlace& pl, int i) {
    b = pl.b;
    off = pl.off;
    const KvShare share(pl.total, p.blocks);
    left = b < 0 ? 0 : share.begin(i + 1) - share.begin(i);
    left_valid = 0;
  }
  // adds a piece to what the block says about its borders
  static __device__ __forceinline__ void note(KvCut& cut, const KvPiece& pc) {
    if (pc.whole) return;
    if ((pc.slot & 1) == 0) {
      cut.flags |= pc.ends ? 6 : 2;
    } else {
      cut.flags |= 1;
      cut.first = pc.s.first;
      cut.head = pc.head;
      cut.row0 = pc.row0;
      cut.rows = pc.rows;
    }
  }
  __device__ __forceinline__ bool next(const KvAttendParams& p, int i, KvPiece& pc) {
    int u, t0, t1;
    do {
      if (left <= 0) return false;
      while (true) {
        if (!left_valid) {
          if (b >= p.kb.batch) return false;
          s = kv_seq<ROWS>(p, b);
          left_valid = 1;
        }
        if (off < kv_seq_work(p, s)) break;
        ++b;
        off = 0;
        left_valid = 0;
      }
      u = (int)kv_div(off, s.tiles);
      const int v0 = (int)(off - (int64_t)u * s.tiles), v1 = (int)min((int64_t)s.tiles, v0 + left);
      off += v1 - v0;
      left -= v1 - v0;
      t0 = max(v0 - kUnitCost<ROWS>, 0);
      t1 = max(v1 - kUnitCost<ROWS>, 0);
    } while (t1 <= t0);                                  // a border within the cost: the next block begins the unit
    const int head = u / s.blocks, rb = kv_row_block(u - head * s.blocks, s.blocks);
    pc.s = s;
    pc.head = head;
    pc.row0 = rb * ROWS;
    pc.rows = min(ROWS, s.new_b * p.group - pc.row0);
    pc.ends = t1 == s.tiles - kUnitCost<ROWS>;
    pc.whole = t0 == 0 && pc.ends;
    pc.slot = 2 * i + (t0 == 0 ? 1 : 0);
    // without a mask nothing behind the last row's own token is seen
    const int t_hi = (pc.row0 + pc.rows - 1) / p.group;
    const int seen = p.mask == nullptr ? min(s.len, s.ctx + t_hi + 1) : s.len;
    pc.t0 = t0;
    pc.t1 = min(t1, (seen + kKvTile - 1) / kKvTile);
    return true;
  }
};

__device__ __forceinline__ float kv_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four 8-bit codes -> two fp16 pairs (bytes 0, 1 and 2, 3), exactly
template <int FMT> __device__ __forceinline__ void kv_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == GL_KV_FP8) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // byte + 128 in the low bits of fp16 1024: 1152 + code
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
// bits 0..3 and 16..19 -> the fp16 pair (code - zero); `zero` holds fp16 1024 + zero twice
__device__ __forceinline__ uint32_t kv_nibbles(uint32_t w, uint32_t zero) {
  uint32_t u = (w & 0x000f000fu) | 0x64006400u;
  const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&u), *reinterpret_cast<__half2*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// two fp32 -> a pair of T
template <typename T> __device__ __forceinline__ uint32_t kv_pair(float a, float b) {
  if constexpr (IsHalf<T>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T, int N> __device__ __forceinline__ void kv_store_n(T* dst, const float (&v)[N]) {
  if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(kv_pair<T>(v[0], v[1]), kv_pair<T>(v[2], v[3]));
  else *reinterpret_cast<uint32_t*>(dst) = kv_pair<T>(v[0], v[1]);
}
template <int N> __device__ __forceinline__ void kv_load_n(const float* src, float (&v)[N]) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
  else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
}
// a / l, rounded once to 16 bits; a row that saw nothing (l = 0) gives zeros
template <typename T> __device__ __forceinline__ void kv_store4(T* dst, float4 a, float l) {
  const float r = l == 0.f ? 0.f : 1.f / l;
  const float v[4] = {l == 0.f ? 0.f : a.x * r, l == 0.f ? 0.f : a.y * r, l == 0.f ? 0.f : a.z * r, l == 0.f ? 0.f : a.w * r};
  kv_store_n<T, 4>(dst, v);
}
#endif
