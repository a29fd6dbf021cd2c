// Paged key-value cache: the append (head norm, position rotation, write) and
// the attention of new tokens over the cached ones.
#include <algorithm>
#include <type_traits>

#include "sg_fp8.cuh"

namespace sg {

namespace attn {

__device__ int g_status = 0;  // first error recorded by a kernel of this unit

__device__ __forceinline__ void record(int code) { atomicCAS(&g_status, 0, code); }

struct Cache {
  uint8_t* k;
  uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  long long page_stride, head_stride, token_stride;  // bytes
  int num_pages, kv_heads, page_shift;
};

// ------------------------------------------------------------------ append
struct AppendArgs {
  Cache c;
  const uint16_t *q, *k, *v;
  long long q_stride, k_stride, v_stride;  // elements between tokens
  int T, q_heads;
  const int32_t* table;  // [table_rows, width]
  int table_rows, width;
  const int32_t* rows;  // [T] or null: token t's table row is t
  const int32_t* positions;
  const float* rope;  // [max_pos, rot]: cos, then sin, of the rot / 2 angles
  int rot, max_pos;
  const uint16_t *q_weight, *k_weight;  // [D] or null
  float eps;
  uint16_t* q_out;  // [T, q_heads, D]
};

// A lane holds two 8-value chunks of a head row that the rotation pairs (or two
// neighbouring ones past the rotated values), D / 16 lanes a row, and the same
// chunks of HPT heads of its token, so cosines and sines are read once for
// them.  Norm sums, the norm and the rotation are in fp32, with one rounding at the
// store; an 8-bit value is value / scale in fp32, rounded to e4m3 (a true division:
// the codes then equal the definition's; the product with 1 / scale is one rounding
// more, which sends middles the wrong way, and makes NaN of zeros where 1 / scale
// overflows, for 33.1 us in place of 36.4 at the size below).
// Bound by latency at decode sizes (one head a lane: as many lanes as there are)
// and at prompt sizes by the bytes of the rows and the lanes in flight for them:
// an 8191-token prompt of 40 heads of 128, in a row of calls, into an 8-bit cache
// 36.4 us (163 MB, 4.4 TB/s) with four heads a lane, two of them loaded ahead, in 80
// registers, and into a bf16 one 34.5 (171 MB, 4.9 TB/s).  Other forms, with the
// product in the 8-bit store, where this one took 33.8: two heads in 64 registers
// 35.1, four loaded at once in 96 41.6, one head 43.5.
template <int D, bool FP8, int HPT>
__global__ void __launch_bounds__(256, 3) append_kv_kernel(const AppendArgs a) {
  constexpr int LP = D / 16;  // lanes per head row
  wait_for_previous();
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  const unsigned groups = (heads + HPT - 1) / HPT;  // a lane's heads are `groups` apart
  const unsigned unit = (blockIdx.x * 256u + threadIdx.x) / LP;
  const int lane = threadIdx.x % LP;
  const unsigned t = unit / groups;
  const int h0 = static_cast<int>(unit - t * groups);
  const bool live = t < static_cast<unsigned>(a.T);
  const int pos = live ? a.positions[t] : -1;
  const bool pos_ok = pos >= 0 && (a.rot == 0 || pos < a.max_pos);
  if (pos >= 0 && !pos_ok) record(SG_ERR_SHAPE);
  const int half = a.rot >> 1;
  const bool turned = lane * 16 < a.rot;
  const int da = turned ? lane * 8 : lane * 16, db = turned ? da + half : da + 8;

  auto load = [&](int i, uint4& xa, uint4& xb) {
    const int head = h0 + i * groups;
    xa = xb = make_uint4(0, 0, 0, 0);
    if (live && head < heads) {
      const int kvh = head < a.q_heads + a.c.kv_heads ? head - a.q_heads : head - a.q_heads - a.c.kv_heads;
      const uint16_t* src = head < a.q_heads ? a.q + t * a.q_stride + head * D
                            : head < a.q_heads + a.c.kv_heads ? a.k + t * a.k_stride + kvh * D
                                                              : a.v + t * a.v_stride + kvh * D;
      xa = ld_stream_v4(src + da);
      xb = ld_stream_v4(src + db);
    }
  };
  uint4 na[2], nb[2];
  load(0, na[0], nb[0]);
  if (HPT > 1) load(1, na[1], nb[1]);
  uint64_t c[4] = {}, sn[4] = {};
  if (turned && pos_ok) {
    const ulonglong2* row = reinterpret_cast<const ulonglong2*>(a.rope + static_cast<long long>(pos) * a.rot + da);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const ulonglong2 u = *(row + i), v = *(row + half / 4 + i);
      c[2 * i] = u.x;
      c[2 * i + 1] = u.y;
      sn[2 * i] = v.x;
      sn[2 * i + 1] = v.y;
    }
  }
  int page = -1;
  if (pos_ok) {
    const int row = a.rows ? a.rows[t] : static_cast<int>(t), col = pos >> a.c.page_shift;
    if (row >= 0 && row < a.table_rows && col < a.width) page = a.table[static_cast<long long>(row) * a.width + col];
    if (page < 0 || page >= a.c.num_pages) {  // nothing is written; the host reads the status
      record(SG_ERR_CAPACITY);
      page = -1;
    }
  }
  const long long place = max(page, 0) * a.c.page_stride + (pos & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int head = h0 + i * groups;
    const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.c.kv_heads;
    uint64_t x[4], y[4];
    unpack8(na[i & 1], x);
    unpack8(nb[i & 1], y);
    if (i + 2 < HPT) load(i + 2, na[i & 1], nb[i & 1]);
    const uint16_t* w = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    if (a.q_weight != nullptr || a.k_weight != nullptr) {  // the same for the whole grid
      uint64_t s2 = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) s2 = f2_fma(x[k], x[k], f2_fma(y[k], y[k], s2));
      float ss = f2_get(s2).x + f2_get(s2).y;
#pragma unroll
      for (int off = LP / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (w != nullptr) {
        const float rstd = rsqrtf(ss / static_cast<float>(D) + a.eps);
        const uint64_t r2 = f2(rstd, rstd);
        uint64_t u[4], v[4];
        unpack8(*(reinterpret_cast<const uint4*>(w + da)), u);
        unpack8(*(reinterpret_cast<const uint4*>(w + db)), v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = f2_mul(x[k], f2_mul(r2, u[k]));
          y[k] = f2_mul(y[k], f2_mul(r2, v[k]));
        }
      }
    }
    if (!live || head >= heads) continue;
    if (turned && pos_ok && !is_v) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t u = f2_fma(y[k] ^ 0x8000000080000000ull, sn[k], f2_mul(x[k], c[k]));  // x c - y s
        y[k] = f2_fma(x[k], sn[k], f2_mul(y[k], c[k]));
        x[k] = u;
      }
    }
    if (is_q) {
      uint16_t* dst = a.q_out + (static_cast<long long>(t) * a.q_heads + head) * D;
      const uint4 zero = make_uint4(0, 0, 0, 0);  // a padding token's
      *reinterpret_cast<uint4*>(dst + da) = pos_ok ? pack8(x) : zero;
      *reinterpret_cast<uint4*>(dst + db) = pos_ok ? pack8(y) : zero;
    } else if (page >= 0) {
      const int kvh = is_v ? head - a.q_heads - a.c.kv_heads : head - a.q_heads;
      uint8_t* dst = (is_v ? a.c.v : a.c.k) + place + kvh * a.c.head_stride;
      if constexpr (FP8) {
        const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[kvh];
        *reinterpret_cast<uint2*>(dst + da) = fp8_pack8(x, scale);
        *reinterpret_cast<uint2*>(dst + db) = fp8_pack8(y, scale);
      } else {
        *reinterpret_cast<uint4*>(dst + da * 2) = pack8(x);
        *reinterpret_cast<uint4*>(dst + db * 2) = pack8(y);
      }
    }
  }
}

// --------------------------------------------------------------- attention
//
// o = softmax(scale q k^T) v of each row's query heads over its cached tokens.
// The query heads that share a key-value head (8 or 16 of them a pass) meet
// every key and value in registers, so the cache is read once for all of them, or
// once for every 16 of a larger group.  Every row of queries reads its tokens by
// itself: made for one or a few new tokens of a sequence; the tokens of a prompt
// work too, each over its whole prefix.  The
// work per cached byte is small (2 to 8 flops), and the kernel is bound by the
// cache's bytes from HBM.  That is why the products run on mma.sync: a tcgen05
// product has at least 64 rows on its token side and keeps its scores in tensor
// memory, two trips away from the softmax, while mma.sync keeps scores, running
// maximum and output in the registers of one warp and has time to spare beside
// the loads.  Tokens (then values of a head) are the 16-row side of each
// product and heads the 8-column side, S^T = K Q^T and O^T = V^T P^T, so that 8
// heads fill it: with heads on the 16-row side half of the work, and of the
// accumulators, was padding (64 unequal rows, 8 heads a group: 131 us so).
//
// A unit of work is a slice: 16 or 32 cached tokens of one (row, key-value head).
// The slices of all rows form one line, which is cut into equal parts, one per
// warp of the (persistent) grid: long and short rows then share the machine
// evenly, whatever the lengths, which only the device knows.  A warp walks its
// part alone (no block-wide barrier): cp.async copies slices ahead of the
// products into its own ring in shared memory, zero-filling tokens past the
// row's length.  Where a warp has a row's slices whole it writes the output;
// otherwise it leaves (running maximum, sum, unscaled output) in the work area,
// and attention_combine_kernel joins the parts in the order of the tokens: the
// result does not depend on timing.  Measured with the joining: 64 rows of 0 to 8192
// tokens, 16 heads over 2 of 256, 90.6 us (537 MB, 0.91 of a copy's rate); one row of
// 131071 50.3 us (0.82); 128 rows of 0 to 8000 over an 8-bit cache, 32 heads over 4
// of 128, 97.2 us (0.83; inputs change from pass to pass here, 93.5 where they stay).

constexpr int WARPS = 4;

struct Args {
  Cache c;
  const uint16_t* q;
  long long q_stride;
  int B, q_heads, group, sub, width;  // sub: parts of at most 16 (8) heads that a group is split into
  const int32_t* table;  // [table_rows, width]
  int table_rows;
  const int32_t* rows;  // [B] or null: row b's table row is b
  const int32_t* lengths;
  int max_length;
  float scale_log2;  // softmax scale * log2(e)
  uint16_t* out;     // [B, q_heads, D]
  int32_t* prefix;   // [B + 1] first slice of each row on the line, then slices per warp
  float2* part_ml;   // [2 * warps][R] running maximum (log2 units) and sum
  float* part_o;     // [2 * warps][R][D]
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
__device__ __forceinline__ uint4 ldsm4_trans(uint32_t a) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
__device__ __forceinline__ float exp2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// four e4m3 bytes to f16: the low two and the high two
__device__ __forceinline__ void e4m3_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// the two values of such a pair
__device__ __forceinline__ void f16_split(uint32_t w, float& lo, float& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.f32.f16 %0, l;\n cvt.f32.f16 %1, h;\n}" : "=f"(lo), "=f"(hi) : "r"(w));
}

// an 8 x 8 matrix of 16-bit values, transposed: lane (g, q) gives row g, columns
// 2q, 2q + 1 and gets column g, rows 2q, 2q + 1
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// c += a b, a [16 x 16] (rows tokens or values), b [16 x 8] (columns heads)
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, bool FP8, bool HALF>
struct Cfg {
  static constexpr int RB = D * (FP8 ? 1 : 2);  // bytes of a cached head row
  // tokens of a slice: narrow rows take 32, so that a slice's fixed work (page,
  // mask, maximum, sums) is spread over as many bytes as a wide row's
  static constexpr int TS = RB <= 128 ? 2 : 1;
  static constexpr int SLICE = 16 * TS;
  static constexpr int KV = SLICE * RB;
  static constexpr int STAGE = 2 * KV;
  // Slices in flight and CTAs per SM, as measured over about 0.5 GB of cache: two
  // slices a warp (one landing, one in use) with as many warps as the registers
  // allow beat three or four slices with fewer warps by 2 to 12 % for rows up to
  // 256 bytes (D 128: 8-bit 90.3 us against 96.2, bf16 87.5 against 91.8; D 64:
  // bf16 84.0 against 87.8, 8-bit 101.8 against 134); rows of 512 bytes leave
  // room for four warps, and three slices each (93.6 us against 95.8).
  static constexpr int STAGES = RB == 512 ? 3 : 2;
  static constexpr int CTAS = RB == 512 ? 1 : D == 256 ? 2 : RB == 64 ? 4 : 3;
  static constexpr int NH = HALF ? 1 : 2;  // groups of 8 heads
  static constexpr int R = 8 * NH;         // heads of a pass
  // 16 heads of 256 values: query fragments and output exceed the registers, and
  // the query fragments stay in shared memory
  static constexpr bool QSMEM = !HALF && D == 256;
  static constexpr int QF = D / 8 * NH;  // query fragment registers
  static constexpr int OFF_Q = WARPS * STAGES * STAGE;
  static constexpr int OFF_MASK = OFF_Q + (QSMEM ? WARPS * QF * 32 * 4 : 0);
  static constexpr int SMEM = OFF_MASK + WARPS * STAGES * 4;
  static_assert((SMEM + 2048) * CTAS <= 228 * 1024, "shared memory budget");
};

// Byte of a 16-byte chunk inside a staged K or V slice.  K is read 16 bytes a
// lane from two rows and four neighbouring chunks at a time, V by ldmatrix from
// eight rows at one chunk: both orders touch all 32 banks.
template <int RB>
__device__ __forceinline__ uint32_t k_at(int row, int chunk) {
  return row * RB + ((RB == 64 ? chunk : chunk ^ ((row & 1) << 2)) << 4);
}
template <int RB>
__device__ __forceinline__ uint32_t v_at(int row, int chunk) {
  return row * RB + ((RB == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) << 4);
}

// A place on the line of slices: row b, head h (of kv_heads * sub), slice k.
struct Cursor {
  int b, h, k, len, slices;
};

__device__ __forceinline__ int table_row(const Args& a, int b) { return a.rows ? a.rows[b] : b; }
__device__ __forceinline__ bool no_row(const Args& a, int b) {
  return a.rows && static_cast<unsigned>(a.rows[b]) >= static_cast<unsigned>(a.table_rows);
}

// Tokens of row b that count; none if it has no row in the table or is longer than allowed.
__device__ __forceinline__ int row_length(const Args& a, int b) {
  const int cap = a.width << a.c.page_shift;
  const int n = a.lengths[b], len = min(max(n, 0), cap);
  return n > a.max_length || no_row(a, b) ? 0 : len;
}

template <int SLICE>
__device__ __forceinline__ void advance(const Args& a, Cursor& c, int heads) {
  if (++c.k < c.slices) return;
  c.k = 0;
  if (++c.h < heads) return;
  c.h = 0;
  do {
    ++c.b;
    c.len = c.b < a.B ? row_length(a, c.b) : SLICE;
    c.slices = (c.len + SLICE - 1) / SLICE;
  } while (c.slices == 0);
}

// What one copy of a slice needs: its head and first token, and in lane t the
// page of token t (-1: past the length, or not a page of the cache).
struct Item {
  int h, tok, page;
};

template <int SLICE>
__device__ __forceinline__ Item fetch(const Args& a, const Cursor& c, int lane) {
  Item it;
  it.h = c.h;
  it.tok = c.k * SLICE;
  it.page = -1;
  const int tok = it.tok + lane % SLICE;
  if (tok < c.len) {
    it.page = *(a.table + static_cast<long long>(table_row(a, c.b)) * a.width + (tok >> a.c.page_shift));
    if (it.page < 0 || it.page >= a.c.num_pages) {  // such tokens are masked; the host reads the status
      record(SG_ERR_CAPACITY);
      it.page = -1;
    }
  }
  return it;
}

template <int D, bool FP8, bool HALF>
__device__ __forceinline__ void issue(const Args& a, const Item& it, int lane, uint32_t stage, uint32_t* mask) {
  using C = Cfg<D, FP8, HALF>;
  constexpr int CPR = C::RB / 16, RPP = 32 / CPR;  // chunks of a row, rows of a pass
  constexpr uint32_t ALL = C::TS == 2 ? 0xffffffffu : 0xffffu;
  const uint32_t live = __ballot_sync(0xffffffffu, it.page >= 0) & ALL;
  if (lane == 0) *mask = live;
  const int chunk = lane % CPR, r0 = lane / CPR;
  const int in_page = (1 << a.c.page_shift) - 1;
  const long long base = (it.h / a.sub) * a.c.head_stride + chunk * 16;
  const long long v_minus_k = a.c.v - a.c.k;
  if (live == ALL && (1 << a.c.page_shift) >= C::SLICE) {  // all in a row of one page
    const int page = __shfl_sync(0xffffffffu, it.page, 0);
    const uint8_t* src = a.c.k + (base + page * a.c.page_stride + ((it.tok & in_page) + r0) * a.c.token_stride);
    const long long step = RPP * a.c.token_stride;
#pragma unroll
    for (int i = 0; i < C::SLICE / RPP; ++i) {
      const int r = r0 + i * RPP;
      cp_async16(stage + k_at<C::RB>(r, chunk), src, 16u);
      cp_async16(stage + C::KV + v_at<C::RB>(r, chunk), src + v_minus_k, 16u);
      src += step;
    }
    return;
  }
#pragma unroll 2
  for (int i = 0; i < C::SLICE / RPP; ++i) {
    const int r = r0 + i * RPP;
    const int page = __shfl_sync(0xffffffffu, it.page, r);
    const uint32_t n = page >= 0 ? 16u : 0u;  // past the row's length: zeros
    const uint8_t* src = a.c.k + (base + max(page, 0) * a.c.page_stride + ((it.tok + r) & in_page) * a.c.token_stride);
    cp_async16(stage + k_at<C::RB>(r, chunk), src, n);
    cp_async16(stage + C::KV + v_at<C::RB>(r, chunk), src + v_minus_k, n);
  }
}

template <int D, bool FP8, bool HALF>
__global__ void __launch_bounds__(WARPS * 32, (Cfg<D, FP8, HALF>::CTAS))
attention_kernel(const Args a) {
  using C = Cfg<D, FP8, HALF>;
  constexpr int RB = C::RB, R = C::R, NH = C::NH, TS = C::TS, SLICE = C::SLICE;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int chunk_pre[WARPS * 32 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;  // row and column pair of a fragment
  const int heads = a.c.kv_heads * a.sub;

  wait_for_previous();
  // the line of slices: each thread counts a run of rows, one scan over the block
  const int run = (a.B + WARPS * 32 - 1) / (WARPS * 32);
  const int b0 = min(static_cast<int>(threadIdx.x) * run, a.B), b1 = min(b0 + run, a.B);
  int n = 0;
  for (int b = b0; b < b1; ++b) n += (row_length(a, b) + SLICE - 1) / SLICE * heads;
  int inc = n;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += o;
  }
  __shared__ int warp_sum[WARPS];
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int excl = before + inc - n;
  chunk_pre[threadIdx.x] = excl;
  const int workers = gridDim.x * WARPS;
  const int per = (total + workers - 1) / workers;
  if (blockIdx.x == 0) {  // for the combining kernel
    int at = excl;
    for (int b = b0; b < b1; ++b) {
      a.prefix[b] = at;
      const int len = a.lengths[b];
      if (len > (a.width << a.c.page_shift)) record(SG_ERR_CAPACITY);
      if (len > 0 && no_row(a, b)) record(SG_ERR_CAPACITY);
      if (len > a.max_length) record(SG_ERR_SHAPE);
      at += (row_length(a, b) + SLICE - 1) / SLICE * heads;
    }
    if (threadIdx.x == 0) a.prefix[a.B] = per;
  }
  __syncthreads();

  // neighbouring parts go to different SMs, so that a short line is spread over all of them
  const int worker = warp * gridDim.x + blockIdx.x;
  const int first = static_cast<int>(min(static_cast<long long>(worker) * per, static_cast<long long>(total)));
  const int last = min(first + per, total);
  if (first >= last) return;

  // the row that holds slice `first`
  int c0 = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    const uint32_t le = __ballot_sync(0xffffffffu, chunk_pre[i * 32 + lane] <= first);
    if (le) c0 = i * 32 + 31 - __clz(le);
  }
  Cursor cur;
  cur.b = min(c0 * run, a.B);
  // several runs may start at the same slice (empty ones): the last of them holds it
  int at = chunk_pre[c0];
  cur.len = row_length(a, cur.b);
  cur.slices = (cur.len + SLICE - 1) / SLICE;
  while (at + cur.slices * heads <= first) {
    at += cur.slices * heads;
    ++cur.b;
    cur.len = row_length(a, cur.b);
    cur.slices = (cur.len + SLICE - 1) / SLICE;
  }
  cur.h = (first - at) / cur.slices;
  cur.k = first - at - cur.h * cur.slices;

  uint32_t* mask = reinterpret_cast<uint32_t*>(smem + C::OFF_MASK) + warp * C::STAGES;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  uint4* q_own = reinterpret_cast<uint4*>(smem + C::OFF_Q) + warp * (C::QF / 4) * 32 + lane;

  Cursor ahead = cur;
  int issued = first;
  {
    Item it[C::STAGES - 1];
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) {
      if (issued + s < last) {
        it[s] = fetch<SLICE>(a, ahead, lane);
        advance<SLICE>(a, ahead, heads);
      }
    }
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) {
      if (issued + s < last) issue<D, FP8, HALF>(a, it[s], lane, ring + s * C::STAGE, mask + s);
      cp_async_commit();
    }
    issued += C::STAGES - 1;
  }
  Item nxt;
  if (issued < last) {
    nxt = fetch<SLICE>(a, ahead, lane);
    advance<SLICE>(a, ahead, heads);
  }

  uint32_t qf[C::QSMEM ? 1 : C::QF];  // per 8 heads: lane (g, q4) holds head g
  float o[D / 16][NH][4];             // lane holds heads 2 q4, 2 q4 + 1 from here on
  float m[NH][2], l[NH][2], sc[NH][2];
  int seg0 = first;  // first slice of the current segment
  bool start = true;
  int slot = 0;
  for (int i = first, st = 0; i < last; ++i) {
    if (start) {
      // A lane takes 16 bytes at a time of a key row (bytes 64 j + 16 q4 ..); the
      // order of a product's inner index is free as long as both sides have the
      // same, so the queries are laid out in that order too.
      const int hv = cur.h / a.sub, s = cur.h - hv * a.sub;
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        const int r = s * R + 8 * t + g;  // head inside its group
        const bool ok = r < a.group;
        const uint16_t* qr = a.q + cur.b * a.q_stride + (static_cast<long long>(hv) * a.group + (ok ? r : 0)) * D;
        sc[t][0] = sc[t][1] = a.scale_log2;
        if constexpr (FP8) {
          // f16 fragments of q / 2^e, 2^e the power of two of the row's largest
          // magnitude: no overflow, exact for bf16 values down to 2^-17 of 2^e, and off
          // by 2^-25 of 2^e at most below that (e4m3 keys are exact in f16, not in a
          // product with bf16 without as many instructions again to widen them)
          float v[D / 64][16];
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < D / 64; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float f[8];
              unpack8(ok ? *(reinterpret_cast<const uint4*>(qr + 64 * j + 16 * q4) + u) : make_uint4(0, 0, 0, 0), f);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                v[j][8 * u + e] = f[e];
                top = fmaxf(top, fabsf(f[e]));
              }
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 1), 253);  // biased exponent
          const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          const float up = __uint_as_float(static_cast<uint32_t>(e) << 23) * a.c.k_scale[hv];
          sc[t][0] *= __shfl_sync(0xffffffffu, up, 8 * q4);  // a lane of head 2 q4
          sc[t][1] *= __shfl_sync(0xffffffffu, up, 8 * q4 + 4);
#pragma unroll
          for (int j = 0; j < D / 64; ++j) {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = f16_pair(v[j][2 * k] * down, v[j][2 * k + 1] * down);
            if constexpr (C::QSMEM) {
              q_own[((j * NH + t) * 2) * 32] = make_uint4(w[0], w[1], w[2], w[3]);
              q_own[((j * NH + t) * 2 + 1) * 32] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) qf[(j * NH + t) * 8 + k] = w[k];
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < RB / 64; ++j) {
            const uint4 w = ok ? *(reinterpret_cast<const uint4*>(qr + 32 * j + 8 * q4)) : make_uint4(0, 0, 0, 0);
            if constexpr (C::QSMEM) {
              q_own[(j * NH + t) * 32] = w;
            } else {
              qf[(j * NH + t) * 4] = w.x;
              qf[(j * NH + t) * 4 + 1] = w.y;
              qf[(j * NH + t) * 4 + 2] = w.z;
              qf[(j * NH + t) * 4 + 3] = w.w;
            }
          }
        }
        m[t][0] = m[t][1] = -3.402823466e38f;
        l[t][0] = l[t][1] = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][t][e] = 0.0f;
      }
      start = false;
    }
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();  // every lane's copies of this slice have landed, and the slice before it is read
    if (issued < last) {
      const int to = st == 0 ? C::STAGES - 1 : st - 1;
      issue<D, FP8, HALF>(a, nxt, lane, ring + to * C::STAGE, mask + to);
      if (++issued < last) {
        nxt = fetch<SLICE>(a, ahead, lane);
        advance<SLICE>(a, ahead, heads);
      }
    }
    cp_async_commit();
    const uint32_t ks = ring + st * C::STAGE, vs = ks + C::KV;
    const uint32_t live = mask[st];

    // scores [16 tokens x 8 heads], TS of them; one alone in two sums, so that the
    // chains of products are half as long
    constexpr int SETS = TS == 1 ? 2 : 1;
    constexpr int QW = FP8 ? 8 : 4;  // query registers of a 64-byte block
    float s2[TS][NH][SETS][4];
#pragma unroll
    for (int x = 0; x < TS * NH * SETS * 4; ++x) (&s2[0][0][0][0])[x] = 0.0f;
#pragma unroll
    for (int j = 0; j < RB / 64; ++j) {
      uint32_t f[NH][QW];
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        if constexpr (C::QSMEM) {
#pragma unroll
          for (int u = 0; u < QW / 4; ++u) {
            const uint4 x = q_own[((j * NH + t) * (QW / 4) + u) * 32];
            f[t][4 * u] = x.x;
            f[t][4 * u + 1] = x.y;
            f[t][4 * u + 2] = x.z;
            f[t][4 * u + 3] = x.w;
          }
        } else {
#pragma unroll
          for (int k = 0; k < QW; ++k) f[t][k] = qf[(j * NH + t) * QW + k];
        }
      }
#pragma unroll
      for (int ts = 0; ts < TS; ++ts) {
        const uint4 k0 = lds128(ks + k_at<RB>(16 * ts + g, 4 * j + q4)), k1 = lds128(ks + k_at<RB>(16 * ts + g + 8, 4 * j + q4));
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int s = 0; s < QW / 2; ++s) {
          uint32_t k[4];
          if constexpr (FP8) {
            e4m3_f16(w0[s], k[0], k[2]);
            e4m3_f16(w1[s], k[1], k[3]);
          } else {
            k[0] = w0[2 * s];
            k[1] = w1[2 * s];
            k[2] = w0[2 * s + 1];
            k[3] = w1[2 * s + 1];
          }
#pragma unroll
          for (int t = 0; t < NH; ++t) mma<FP8>(s2[ts][t][s % SETS], k, f[t][2 * s], f[t][2 * s + 1]);
        }
      }
    }

    // running softmax in log2 units; masked tokens score -inf, and the maximum
    // never falls below the lowest finite value, so no difference is inf - inf
    uint32_t ph[TS][NH][2], pl[TS][NH][2];  // probabilities, tokens 2 q4 .. of head g, and tokens + 8
    float alpha[NH][2];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < NH; ++t) {
      float p[TS][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v[TS][2], top = m[t][e];
#pragma unroll
        for (int ts = 0; ts < TS; ++ts)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float sum = s2[ts][t][0][2 * x + e];
            if constexpr (SETS == 2) sum += s2[ts][t][SETS - 1][2 * x + e];
            v[ts][x] = (live >> (16 * ts + 8 * x + g)) & 1 ? sum * sc[t][e] : -INFINITY;
            top = fmaxf(top, v[ts][x]);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        alpha[t][e] = exp2_(m[t][e] - top);
        moved = moved || m[t][e] != top;
        m[t][e] = top;
        // f16 parts carry 2^13, so that their sum keeps 22 bits down to 2^-16, and the
        // first alone eleven down to 2^-27
        const float shift = FP8 ? top - 13.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int ts = 0; ts < TS; ++ts) {
          p[ts][e] = exp2_(v[ts][0] - shift);
          p[ts][2 + e] = exp2_(v[ts][1] - shift);
          sum += p[ts][e] + p[ts][2 + e];
        }
        l[t][e] = l[t][e] * alpha[t][e] + sum;
      }
#pragma unroll
      for (int ts = 0; ts < TS; ++ts)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          // in two parts: one part alone (bf16 8 bits, f16 11) would round as much as the
          // output does, or an eighth of it.  Over an 8-bit cache the second part costs 1 %
          // where 8 heads share a key (128 rows of 0 to 8000 tokens, 32 heads over 4 of
          // 128, 92.4 -> 93.5 us) and 7 to 14 % where 16 do (64 rows of 0 to 8192, 16 over
          // 1 of 128, 25.2 -> 28.8)
          const float p0 = p[ts][2 * x], p1 = p[ts][2 * x + 1];
          if constexpr (FP8) {
            float h0, h1;
            const uint32_t hi = f16_pair(p0, p1);
            f16_split(hi, h0, h1);
            ph[ts][t][x] = transpose8(hi);
            pl[ts][t][x] = transpose8(f16_pair(p0 - h0, p1 - h1));
          } else {
            const uint32_t hi = bf16_pair(p0, p1);
            ph[ts][t][x] = transpose8(hi);
            pl[ts][t][x] = transpose8(bf16_pair(p0 - lo_bf16(hi), p1 - hi_bf16(hi)));
          }
        }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int t = 0; t < NH; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][t][e] *= alpha[t][e & 1];
    }

    if constexpr (FP8) {
      // a transposed 16-bit cell holds values 2n, 2n + 1 of a token: rows 0..7 of
      // a 16-value product are a chunk's even values, rows 8..15 its odd ones
      const int vrow = lane & 15, vchunk = lane >> 4;
#pragma unroll
      for (int c = 0; c < RB / 16; c += 2) {
#pragma unroll
        for (int ts = 0; ts < TS; ++ts) {
          const uint4 v = ldsm4_trans(vs + v_at<RB>(16 * ts + vrow, c + vchunk));
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
          uint32_t f[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            e4m3_f16(__byte_perm(w[2 * u], 0, 0x3120), f[u][0], f[u][1]);
            e4m3_f16(__byte_perm(w[2 * u + 1], 0, 0x3120), f[u][2], f[u][3]);
          }
#pragma unroll
          for (int t = 0; t < NH; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) mma<true>(o[c + u][t], f[u], ph[ts][t][0], ph[ts][t][1]);
#pragma unroll
          for (int t = 0; t < NH; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) mma<true>(o[c + u][t], f[u], pl[ts][t][0], pl[ts][t][1]);
        }
      }
    } else {
      const int vrow = (lane & 7) + (lane >> 4) * 8, vchunk = (lane >> 3) & 1;
#pragma unroll
      for (int c = 0; c < RB / 16; c += 4) {
#pragma unroll
        for (int ts = 0; ts < TS; ++ts) {
          const uint4 v0 = ldsm4_trans(vs + v_at<RB>(16 * ts + vrow, c + vchunk));
          const uint4 v1 = ldsm4_trans(vs + v_at<RB>(16 * ts + vrow, c + 2 + vchunk));
          const uint32_t f0[4] = {v0.x, v0.y, v0.z, v0.w}, f1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
          for (int t = 0; t < NH; ++t) {
            mma<false>(o[c / 2][t], f0, ph[ts][t][0], ph[ts][t][1]);
            mma<false>(o[c / 2 + 1][t], f1, ph[ts][t][0], ph[ts][t][1]);
          }
#pragma unroll
          for (int t = 0; t < NH; ++t) {
            mma<false>(o[c / 2][t], f0, pl[ts][t][0], pl[ts][t][1]);
            mma<false>(o[c / 2 + 1][t], f1, pl[ts][t][0], pl[ts][t][1]);
          }
        }
      }
    }
    if (++st == C::STAGES) st = 0;

    if (cur.k + 1 == cur.slices || i + 1 == last) {  // the segment ends here
      const int hv = cur.h / a.sub, s = cur.h - hv * a.sub;
      const bool whole = cur.k + 1 == cur.slices && i + 1 - seg0 == cur.slices;
      const float vscale = FP8 ? a.c.v_scale[hv] : 1.0f;
#pragma unroll
      for (int t = 0; t < NH; ++t) {
        float sum[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sum[e] = l[t][e];
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], off);
        }
        const int r = 8 * t + 2 * q4;  // this lane's heads of the pass: r, r + 1
        if (whole) {
          float inv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)  // no token counts: zeros; NaN stays
            inv[e] = sum[e] > 0.0f ? vscale / sum[e] : sum[e] == 0.0f ? 0.0f : sum[e];
          const int head = s * R + 8 * t + g;  // after the transposition a lane has head g
          uint16_t* dst = a.out + (static_cast<long long>(cur.b) * a.q_heads + static_cast<long long>(hv) * a.group + head) * D;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const uint32_t x = transpose8(bf16_pair(o[d][t][0] * inv[0], o[d][t][1] * inv[1]));
            const uint32_t y = transpose8(bf16_pair(o[d][t][2] * inv[0], o[d][t][3] * inv[1]));
            if (head < a.group) {
              if constexpr (FP8) {  // x: even values, y: odd ones
                *reinterpret_cast<uint2*>(dst + 16 * d + 4 * q4) = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
              } else {
                *reinterpret_cast<uint32_t*>(dst + 16 * d + 2 * q4) = x;
                *reinterpret_cast<uint32_t*>(dst + 16 * d + 8 + 2 * q4) = y;
              }
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (s * R + r + e >= a.group) continue;
            const long long ps = (2LL * worker + slot) * R + r + e;
            if (g == 0) a.part_ml[ps] = make_float2(m[t][e], sum[e]);
            float* dst = a.part_o + ps * D;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              if constexpr (FP8) {
                *reinterpret_cast<float2*>(dst + 16 * d + 2 * g) = make_float2(o[d][t][e] * vscale, o[d][t][2 + e] * vscale);
              } else {
                dst[16 * d + g] = o[d][t][e];
                dst[16 * d + 8 + g] = o[d][t][2 + e];
              }
            }
          }
        }
      }
      seg0 = i + 1;
      slot = 1;  // a later incomplete segment is the warp's last
      start = true;
    }
    advance<SLICE>(a, cur, heads);
  }
}

// Joins the parts that the warps left of a (row, head), in the order of the
// tokens; rows without tokens become zeros.  A group of PIECE / 4 lanes (four
// values each) walks the parts of PIECE values of one head.  The kernel is a chain
// of a few L2 latencies: few (row, head)s may have hundreds of parts each (one long
// row over the whole grid), and a block's GROUPS groups walk a share each, joined in
// shared memory; many have few parts each, and one group walks them all (GROUPS 1).
// How many parts a row really has, only the device knows: the host goes by the number
// of (row, head)s, as if all rows were equally long.  One long row among many short ones
// is joined by one group, four parts at a time.
template <int D, int R, int SLICE, int PIECE, int GROUPS>
__global__ void __launch_bounds__(GROUPS == 1 ? 128 : PIECE / 4 * GROUPS)
attention_combine_kernel(const Args a) {
  constexpr int LANES = PIECE / 4, PIECES = D / PIECE;
  __shared__ float4 acc_s[GROUPS][LANES];
  __shared__ float2 ml_s[GROUPS];
  wait_for_previous();
  const int group = GROUPS == 1 ? 0 : threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const long long unit = GROUPS == 1 ? (static_cast<long long>(blockIdx.x) * 128 + threadIdx.x) / LANES : blockIdx.x;
  const long long row = unit / PIECES;
  if (row >= static_cast<long long>(a.B) * a.q_heads) return;
  const int d = static_cast<int>(unit - row * PIECES) * PIECE + lane * 4;
  const int b = static_cast<int>(row / a.q_heads), hq = static_cast<int>(row - static_cast<long long>(b) * a.q_heads);
  const int hv = hq / a.group, rest = hq - hv * a.group;
  const int per = a.prefix[a.B], at = a.prefix[b];  // with the length: one latency
  const int slices = (row_length(a, b) + SLICE - 1) / SLICE;
  uint2* dst = reinterpret_cast<uint2*>(a.out + row * D + d);
  if (slices == 0) {
    if (group == 0) *dst = make_uint2(0, 0);
    return;
  }
  const int s = at + (hv * a.sub + rest / R) * slices;
  const int w0 = s / per, w1 = (s + slices - 1) / per;
  if (w0 == w1) return;  // one warp had the whole and wrote it
  float m = -3.402823466e38f, l = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 4;  // parts in flight
  for (int w = w0 + group; w <= w1; w += U * GROUPS) {
    float2 ml[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = min(w + u * GROUPS, w1);  // past the end: the last part again, left out below
      const int slot = x == w0 && x * per < s ? 1 : 0;
      const long long ps = (2LL * x + slot) * R + rest % R;
      ml[u] = __ldcg(a.part_ml + ps);
      v[u] = __ldcg(reinterpret_cast<const float4*>(a.part_o + ps * D + d));
      if (w + u * GROUPS > w1) ml[u] = make_float2(-3.402823466e38f, 0.0f), v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float top = fmaxf(m, ml[u].x);
      const float x = exp2_(m - top), y = exp2_(ml[u].x - top);
      m = top;
      l = l * x + ml[u].y * y;
      o = make_float4(o.x * x + v[u].x * y, o.y * x + v[u].y * y, o.z * x + v[u].z * y, o.w * x + v[u].w * y);
    }
  }
  if constexpr (GROUPS > 1) {
    acc_s[group][lane] = o;
    if (lane == 0) ml_s[group] = make_float2(m, l);
    __syncthreads();
    if (group != 0) return;
    float top = m;
    for (int w = 1; w < GROUPS; ++w) top = fmaxf(top, ml_s[w].x);
    l = 0.0f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < GROUPS; ++w) {
      const float y = exp2_(ml_s[w].x - top);
      const float4 v = acc_s[w][lane];
      l += ml_s[w].y * y;
      o = make_float4(o.x + v.x * y, o.y + v.y * y, o.z + v.z * y, o.w + v.w * y);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  *dst = make_uint2(bf16_pair(o.x * inv, o.y * inv), bf16_pair(o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ host side
static int num_sms(int dev) {
  static int n[64] = {};
  if (n[dev] == 0) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] > 0 ? n[dev] : 148;
}

static bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

static int check_cache(const sg_kv_cache* c, Cache* out) {
  if (!c) return SG_ERR_INVALID_ARG;
  if (c->bits != 16 && c->bits != 8) return SG_ERR_FORMAT;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return SG_ERR_SHAPE;
  if (c->num_pages < 1 || c->kv_heads < 1 || c->page_size < 1 || c->page_size > (1 << 20) ||
      (c->page_size & (c->page_size - 1)))
    return SG_ERR_SHAPE;
  const int eb = c->bits / 8;
  if ((c->page_stride * eb) % 16 || (c->head_stride * eb) % 16 || (c->token_stride * eb) % 16) return SG_ERR_SHAPE;
  if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0) return SG_ERR_SHAPE;
  if (!c->k || !c->v || misaligned16(c->k) || misaligned16(c->v)) return SG_ERR_INVALID_ARG;
  if (c->bits == 8 && (!c->k_scale || !c->v_scale)) return SG_ERR_INVALID_ARG;
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->page_stride = c->page_stride * eb;
  out->head_stride = c->head_stride * eb;
  out->token_stride = c->token_stride * eb;
  out->num_pages = c->num_pages;
  out->kv_heads = c->kv_heads;
  out->page_shift = 0;
  while ((1 << out->page_shift) < c->page_size) ++out->page_shift;
  return SG_OK;
}

// Where a call's parts go in the work area (bytes); the grid is the device's
struct Work {
  int grid, workers, rows;
  long long off_ml, off_o, bytes;
};

template <int D, bool FP8, bool HALF>
static Work work_layout(int dev, int B) {
  using C = Cfg<D, FP8, HALF>;
  Work w;
  w.grid = num_sms(dev) * C::CTAS;
  w.workers = w.grid * WARPS;
  w.rows = C::R;
  w.off_ml = (static_cast<long long>(B + 1) * 4 + 255) / 256 * 256;
  w.off_o = w.off_ml + (2LL * w.workers * C::R * 8 + 255) / 256 * 256;
  w.bytes = w.off_o + 2LL * w.workers * C::R * D * 4;
  return w;
}

template <int D, int R, int SLICE, int PIECE, int GROUPS>
static int launch_combine(const Args& a, cudaStream_t s) {
  const long long units = static_cast<long long>(a.B) * a.q_heads * (D / PIECE);
  SG_CUDA_TRY(launch_after_previous(attention_combine_kernel<D, R, SLICE, PIECE, GROUPS>,
                                    static_cast<unsigned>(GROUPS == 1 ? (units * (PIECE / 4) + 127) / 128 : units),
                                    GROUPS == 1 ? 128 : PIECE / 4 * GROUPS, 0, s, a));
  return SG_OK;
}

template <int D, bool FP8, bool HALF>
static int launch_attention(Args a, uint8_t* work, int dev, cudaStream_t s) {
  using C = Cfg<D, FP8, HALF>;
  const Work w = work_layout<D, FP8, HALF>(dev, a.B);
  a.prefix = reinterpret_cast<int32_t*>(work);
  a.part_ml = reinterpret_cast<float2*>(work + w.off_ml);
  a.part_o = reinterpret_cast<float*>(work + w.off_o);
  a.sub = (a.group + C::R - 1) / C::R;
  static bool attr_done[64] = {};
  if (!attr_done[dev]) {
    SG_CUDA_TRY(cudaFuncSetAttribute(attention_kernel<D, FP8, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_done[dev] = true;
  }
  SG_CUDA_TRY(launch_after_previous(attention_kernel<D, FP8, HALF>, w.grid, WARPS * 32, C::SMEM, s, a));
  // us with the joining, 32 groups / 16 / 4 / 1, by (row, head)s: 16 of 131071 tokens 49 /
  // 51 / 77 / 160; 128 of 0 to 20000 16.2 / 16.8 / 31 / 81; 256 of 0 to 600 10.0 / 7.7 / 9.6
  // / 20; 512 of 0 to 4000 22 / 16.5 / 17.9 / 31 (heads of 256 45 / 36 / 32 / 39); 1024 of 0
  // to 8192 119 / 100 / 91 / 94; 2048 of 0 to 600 41 / 23 / 14.5 / 16.7; 4096 of 0 to 8000
  // 153 / 113 / 96 / 94; 16384 of 0 to 1000 304 / 168 / 106 / 94.
  const long long rows = static_cast<long long>(a.B) * a.q_heads;
  constexpr int PIECE = D < 128 ? D : 128;
  if (rows <= 64) return launch_combine<D, C::R, C::SLICE, 32, 32>(a, s);
  if (rows <= 512) return launch_combine<D, C::R, C::SLICE, 32, 16>(a, s);
  if (rows <= 2048) return launch_combine<D, C::R, C::SLICE, PIECE, 4>(a, s);
  return launch_combine<D, C::R, C::SLICE, PIECE, 1>(a, s);
}

template <typename F>
static int by_format(int head_dim, int bits, bool half, F f) {
  switch (head_dim * 100 + bits * 2 + (half ? 1 : 0)) {
    case 6432: return f(std::integral_constant<int, 64>(), std::false_type(), std::false_type());
    case 6433: return f(std::integral_constant<int, 64>(), std::false_type(), std::true_type());
    case 6416: return f(std::integral_constant<int, 64>(), std::true_type(), std::false_type());
    case 6417: return f(std::integral_constant<int, 64>(), std::true_type(), std::true_type());
    case 12832: return f(std::integral_constant<int, 128>(), std::false_type(), std::false_type());
    case 12833: return f(std::integral_constant<int, 128>(), std::false_type(), std::true_type());
    case 12816: return f(std::integral_constant<int, 128>(), std::true_type(), std::false_type());
    case 12817: return f(std::integral_constant<int, 128>(), std::true_type(), std::true_type());
    case 25632: return f(std::integral_constant<int, 256>(), std::false_type(), std::false_type());
    case 25633: return f(std::integral_constant<int, 256>(), std::false_type(), std::true_type());
    case 25616: return f(std::integral_constant<int, 256>(), std::true_type(), std::false_type());
    case 25617: return f(std::integral_constant<int, 256>(), std::true_type(), std::true_type());
    default: return SG_ERR_SHAPE;
  }
}

}  // namespace attn

int attn_device_status(int reset) {
  int v = 0;
  SG_CUDA_TRY(cudaMemcpyFromSymbol(&v, attn::g_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    SG_CUDA_TRY(cudaMemcpyToSymbol(attn::g_status, &zero, sizeof(int)));
  }
  return v;
}

}  // namespace sg

extern "C" int sg_append_kv(const sg_kv_cache* cache, const uint16_t* q, long long q_stride, const uint16_t* k,
                            long long k_stride, const uint16_t* v, long long v_stride, int T, int q_heads,
                            const int32_t* page_table, int table_rows, int table_width, const int32_t* rows,
                            const int32_t* positions, const float* rope, int rot, int max_pos,
                            const uint16_t* q_weight, const uint16_t* k_weight, float eps, uint16_t* q_out,
                            void* stream) {
  using namespace sg::attn;
  AppendArgs a{};
  const int st = check_cache(cache, &a.c);
  if (st != SG_OK) return st;
  const int D = cache->head_dim;
  if (T < 0 || q_heads < 0 || table_rows < 0 || table_width < 0 || rot < 0) return SG_ERR_INVALID_ARG;
  if (rot % 16 || rot > D || q_stride % 8 || k_stride % 8 || v_stride % 8) return SG_ERR_SHAPE;
  if (q_stride < 0 || k_stride < 0 || v_stride < 0) return SG_ERR_SHAPE;
  if (T == 0) return SG_OK;
  if (!k || !v || !positions || !page_table || (q_heads > 0 && (!q || !q_out))) return SG_ERR_INVALID_ARG;
  if (rot > 0 && (!rope || max_pos < 1)) return SG_ERR_INVALID_ARG;
  if (misaligned16(q) || misaligned16(k) || misaligned16(v) || misaligned16(rope) || misaligned16(q_weight) ||
      misaligned16(k_weight) || misaligned16(q_out))
    return SG_ERR_INVALID_ARG;
  a.q = q; a.k = k; a.v = v;
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.T = T; a.q_heads = q_heads;
  a.table = page_table; a.table_rows = table_rows; a.width = table_width;
  a.rows = rows; a.positions = positions;
  a.rope = rope; a.rot = rot; a.max_pos = max_pos;
  a.q_weight = q_weight; a.k_weight = k_weight; a.eps = eps; a.q_out = q_out;
  const long long heads = q_heads + 2LL * a.c.kv_heads;
  int dev = 0;
  SG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return SG_ERR_CUDA;
  // four heads a lane once that still leaves every SM its fill of lanes
  const bool four = T * heads * (D / 16) >= 4LL * num_sms(dev) * 768;
  const long long blocks = (T * (four ? (heads + 3) / 4 : heads) * (D / 16) + 255) / 256;
  if (blocks > (1 << 23)) return SG_ERR_SHAPE;
  return by_format(D, cache->bits, false, [&](auto dim, auto fp8, auto) -> int {
    SG_CUDA_TRY(sg::launch_after_previous(four ? append_kv_kernel<dim.value, fp8.value, 4> : append_kv_kernel<dim.value, fp8.value, 1>,
                                      (unsigned)blocks, 256, 0, (cudaStream_t)stream, a));
    return SG_OK;
  });
}

extern "C" long long sg_paged_attention_work_bytes(const sg_kv_cache* cache, int B, int q_heads) {
  using namespace sg::attn;
  Cache c;
  const int st = check_cache(cache, &c);
  if (st != SG_OK) return st;
  if (B < 0 || q_heads < 1) return SG_ERR_INVALID_ARG;
  if (q_heads % c.kv_heads) return SG_ERR_SHAPE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();  // no device: the size for the card this library is built for
    dev = 0;
  }
  if (dev < 0 || dev >= 64) return SG_ERR_CUDA;
  long long bytes = 0;
  const int rc = by_format(cache->head_dim, cache->bits, q_heads / c.kv_heads <= 8, [&](auto dim, auto fp8, auto half) -> int {
    bytes = work_layout<dim.value, fp8.value, half.value>(dev, B).bytes;
    return SG_OK;
  });
  return rc == SG_OK ? bytes : rc;
}

extern "C" int sg_paged_attention_rows(const sg_kv_cache* cache, const uint16_t* q, long long q_stride, int B, int q_heads,
                                       const int32_t* page_table, int table_rows, int table_width, const int32_t* rows,
                                       const int32_t* lengths, int max_length, float scale, uint16_t* out, void* work,
                                       long long work_bytes, void* stream) {
  using namespace sg::attn;
  const long long need = sg_paged_attention_work_bytes(cache, B, q_heads);
  if (need < 0) return (int)need;
  Args a{};
  check_cache(cache, &a.c);
  if (table_rows < 0 || table_width < 0 || max_length < 0) return SG_ERR_INVALID_ARG;
  if (q_stride % 8 || q_stride < 0) return SG_ERR_SHAPE;
  if (!rows && table_rows < B) return SG_ERR_INVALID_ARG;
  if (B == 0) return SG_OK;
  if (!q || !lengths || !out || !work || (table_rows > 0 && table_width > 0 && !page_table)) return SG_ERR_INVALID_ARG;
  if (misaligned16(q) || misaligned16(out) || misaligned16(work)) return SG_ERR_INVALID_ARG;
  if (work_bytes < need) return SG_ERR_CAPACITY;
  a.group = q_heads / a.c.kv_heads;
  const bool half = a.group <= 8;
  const long long heads = static_cast<long long>(a.c.kv_heads) * ((a.group + (half ? 7 : 15)) / (half ? 8 : 16));
  const long long longest = static_cast<long long>(table_width) << a.c.page_shift;
  const long long slices = heads * ((longest + 15) / 16);  // of a row, at most
  if (longest > (1 << 30) || slices > (1 << 30)) return SG_ERR_SHAPE;
  a.q = q; a.q_stride = q_stride; a.q_heads = q_heads; a.width = table_width;
  a.table = page_table; a.table_rows = table_rows; a.rows = rows; a.lengths = lengths; a.max_length = max_length; a.scale_log2 = scale * 1.44269504f; a.out = out;
  int dev = 0;
  SG_CUDA_TRY(cudaGetDevice(&dev));
  // A line's slices are counted in 32 bits: where the table could hold more, as many
  // rows at a time as fit, one after the other over the same work area.
  const int most = static_cast<int>(std::min<long long>(B, (1 << 30) / std::max<long long>(slices, 1)));
  return by_format(cache->head_dim, cache->bits, half, [&](auto dim, auto fp8, auto hf) -> int {
    for (int b = 0; b < B; b += a.B) {
      a.B = std::min(most, B - b);
      const int st = launch_attention<dim.value, fp8.value, hf.value>(a, static_cast<uint8_t*>(work), dev, (cudaStream_t)stream);
      if (st != SG_OK) return st;
      a.q += a.B * q_stride;
      a.out += static_cast<long long>(a.B) * q_heads * dim.value;
      a.lengths += a.B;
      if (rows) {
        a.rows += a.B;
      } else {
        a.table += static_cast<long long>(a.B) * table_width;
        a.table_rows -= a.B;
      }
    }
    return SG_OK;
  });
}

extern "C" int sg_paged_attention(const sg_kv_cache* cache, const uint16_t* q, long long q_stride, int B, int q_heads,
                                  const int32_t* page_table, int table_width, const int32_t* lengths, float scale,
                                  uint16_t* out, void* work, long long work_bytes, void* stream) {
  return sg_paged_attention_rows(cache, q, q_stride, B, q_heads, page_table, B, table_width, nullptr, lengths, INT32_MAX, scale,
                                 out, work, work_bytes, stream);
}
