// Matrix product of e4m3 rows and e4m3 weights with fp32 scales per block of
// 128, on the 5th-generation tensor cores.
//
// out[t, n] = sum_b sx[b, t] sw[n / 128, b] (sum_{k in b} x8[t, k] w8[n, k]).
// The scales differ from block to block along k, so the products of one block
// are summed by the tensor cores in tensor memory (four tcgen05.mma of 32
// values, fp32), and the blocks in the registers of the epilogue warps: each
// reads the block's accumulator and adds scale * accumulator.  A ring of
// accumulators keeps the tensor cores going meanwhile.
//
// The product's 128-row side is the tensor memory lanes, its other side (BN) the
// columns.  Two forms:
//  - TM (tokens on the 128-row side, 65 tokens and more): a lane is a token and
//    the columns are weight rows, so a lane's scale is one number for 128
//    columns: sx of its token times sw of the columns' block (with weights on the
//    lanes, each of 256 columns has a scale of its own, and reading them from
//    shared memory for every block took twice the tensor cores' time: 4096 x 4096
//    x 9216 324 us).
//  - weights on the 128-row side (up to 64 tokens): a single token costs 16
//    columns, not 128 rows.
// Operands are TMA boxes of 128 bytes of k (SW128; what lies past the ends is the
// TMA's zero fill).
//
// Warp roles: w0 TMA producer; w1 tensor memory and MMA issue; w2, w3 scales (the
// products sx * sw of a block, ahead, into a ring in shared memory); w4.. epilogue,
// one TMEM lane quadrant each.
//
// Where tiles are fewer than SMs, a cluster shares one tile, each of its CTAs a
// range of k blocks, and the partial sums are added in rank order through
// distributed shared memory.
//
// Bound by the weights' bytes and a chain of latencies for few tokens (16 x 2048 x
// 5120 6.4 us in a row of calls, 1.6 of it bytes), by the tensor cores and the
// epilogue beside them for many (4096 x 4096 x 9216 152 us, 2.03 PFLOP/s, in a
// short burst; 174 at the card's power cap).
//
// Every mbarrier wait is bounded; on expiry the CTA records SG_ERR_TIMEOUT, waits
// (bounded) for its copies in flight, frees its tensor memory and returns.
#include "sg_fp8.cuh"
#include "sg_tc.cuh"

namespace sg {

namespace f8 {

using namespace tc;

constexpr int BM = 128;  // rows of a tile
constexpr int BK = 128;  // bytes of k per stage: one block, one 128-byte swizzle row
constexpr int EPI_WARP0 = 4;

// BN: columns of a tile (weights on the rows: any multiple of 16 up to BN)
template <bool TM, int BN>
struct Cfg {
  static constexpr int A_BYTES = BM * BK;
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int CTAS = BN <= 64 ? 2 : 1;  // per SM
  static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : BN == 128 ? 6 : 4;
  static constexpr int EW = BN <= 64 ? 4 : 8;  // epilogue warps: 4 lane quadrants x 1 or 2 column groups
  static constexpr int CH = BN < 32 ? 16 : 32;  // columns of one tensor memory load
  static constexpr int CHUNKS = BN / CH * 4 / EW;  // loads per epilogue thread and block
  static constexpr int NACC = BN == 256 ? 2 : BN <= 32 ? 8 : 4;
  static constexpr int TMEM_COLS = NACC * BN;
  // scale ring: a block's products sx * sw, one for each column, or (TM) for each
  // row and block of weight rows
  static constexpr int SU = TM ? 4 : 8;  // blocks handed over at a time
  static constexpr int SR = 2;  // of those
  static constexpr int SW = TM ? BM * (BN > BM ? 2 : 1) : BN;
  static constexpr int THREADS = (EPI_WARP0 + EW) * 32;
  static constexpr int OFF_S = STAGES * STAGE;
  // TM: a place of 32 rows x 32 bf16 per epilogue warp, through which a tile leaves
  // as whole pieces of rows (rows 80 bytes apart: no bank conflicts)
  static constexpr int OUT_PITCH = 80;
  static constexpr int OUT_PLACE = TM ? 32 * OUT_PITCH : 0;
  static constexpr int OFF_O = OFF_S + SR * SU * SW * 4;
  static constexpr int OFF_BAR = OFF_O + EW * OUT_PLACE;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * NACC + 2 * SR;
  static constexpr int SMEM = OFF_BAR + NUM_BARS * 8 + 16 + 1024;
  static_assert((SMEM + 1024) * CTAS <= 228 * 1024, "shared memory budget");
  static_assert(TMEM_COLS * CTAS <= 512 && TMEM_COLS >= 32, "tensor memory budget");
  static constexpr int PITCH = TM ? BN + 4 : BM;  // floats between rows (TM: tokens, else columns) of partial sums
  static_assert(PITCH * (TM ? BM : BN) * 4 <= STAGES * STAGE, "partial sums reuse the operand ring");
  // TM: an epilogue thread holds 64 or 128 sums and two loads of 32 columns; the
  // first four warps give up registers for it, in all what the launch has (128 x 56
  // + 256 x 224 = 384 x 168; 128 x 56 + 128 x 200 = 256 x 128)
  static constexpr int REGS = !TM ? 0 : BN == 256 ? 224 : BN == 64 ? 200 : 0;
};

struct Args {
  const float* sx;
  const float* sw;
  uint16_t* out;
  int T, N, KB;  // KB: blocks of k
  int MT, NT;    // tiles along the rows / the columns
  int bn, split;
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
      ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // does not wait
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// 16 or 32 accumulator columns of this warp's lanes, complete on return
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// the same load without the wait, and the wait that makes r usable
__device__ __forceinline__ void tmem_issue(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// acc += d * s over 32 columns
__device__ __forceinline__ void add_scaled(unsigned long long (&acc)[16], const uint32_t (&d)[32], float s) {
  unsigned long long s2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const unsigned long long v = static_cast<unsigned long long>(d[2 * j + 1]) << 32 | d[2 * j];
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[j]) : "l"(v), "l"(s2));
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, int rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <bool TM, int BN>
__global__ void __launch_bounds__(Cfg<TM, BN>::THREADS, Cfg<TM, BN>::CTAS)
fp8_linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args args) {
  using C = Cfg<TM, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* scales = reinterpret_cast<float*>(smem + C::OFF_S);  // [SR][SU][SW]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                 // [STAGES] operands landed (TMA)
  uint64_t* empty = full + C::STAGES;    // [STAGES] operands read (MMA commit)
  uint64_t* acc_full = empty + C::STAGES;     // [NACC] block's products complete (MMA commit)
  uint64_t* acc_empty = acc_full + C::NACC;   // [NACC] read by the epilogue warps
  uint64_t* s_full = acc_empty + C::NACC;     // [SR] SU blocks' scales written
  uint64_t* s_empty = s_full + C::SR;         // [SR] read by the epilogue warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const Ctl ctl{abort_flag};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::NACC; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], C::EW);
    }
    for (int i = 0; i < C::SR; ++i) {
      mbar_init(&s_full[i], 2);
      mbar_init(&s_empty[i], C::EW);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_previous();
  asm volatile("fence.proxy.async.global;" ::: "memory");  // what the kernel before wrote, for the TMA loads

  // this CTA's tiles, and its range of k blocks of each
  const int split = args.split, bn = args.bn;
  const int rank = split > 1 ? blockIdx.x % split : 0;
  const int tile0 = blockIdx.x / split, tiles = args.MT * args.NT, step = gridDim.x / split;
  const int kb0 = static_cast<int>(static_cast<long long>(args.KB) * rank / split);
  const int kb1 = static_cast<int>(static_cast<long long>(args.KB) * (rank + 1) / split);

  if (warp < EPI_WARP0) {
    if constexpr (C::REGS > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0) {
        const uint32_t bytes = C::A_BYTES + bn * BK;
        int st = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = tile0; t < tiles && ok; t += step) {
          const int m = t % args.MT, n = t / args.MT;
          for (int kb = kb0; kb < kb1; ++kb) {
            ok = wait_bar(&empty[st], ph ^ 1, ctl);
            if (!ok) break;
            uint8_t* dst = smem + st * C::STAGE;
            mbar_expect_tx(&full[st], bytes);
            tma_load_2d(dst, &tmA, kb * BK, m * BM, &full[st]);
            tma_load_2d(dst + C::A_BYTES, &tmB, kb * BK, n * bn, &full[st]);
            ++issued;
            if (++st == C::STAGES) { st = 0; ph ^= 1; }
          }
        }
        if (!ok) {  // wait for the copies still in flight (bounded)
          for (int i = 0; i < min(issued, C::STAGES); ++i) {
            int s = st - 1 - i;
            uint32_t p = ph;
            if (s < 0) { s += C::STAGES; p ^= 1; }
            const long long t0 = clock64();
            while (!mbar_try_wait(&full[s], p) && clock64() - t0 < WAIT_CYCLES) {
            }
          }
        }
      }
    } else if (warp == 1) {
      if (lane == 0) {
        // D fp32, A and B e4m3, both K-major, M = 128, N = bn
        const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(bn >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
        int st = 0, ab = 0;
        uint32_t ph = 0, ap = 0;
        bool ok = true;
        for (int t = tile0; t < tiles && ok; t += step) {
          for (int kb = kb0; kb < kb1; ++kb) {
            ok = wait_bar(&acc_empty[ab], ap ^ 1, ctl);
            ok = ok && wait_bar(&full[st], ph, ctl);
            if (!ok) break;
            tc_fence_after();
            const uint64_t a = desc_sw128(smem_u32(smem + st * C::STAGE));
            const uint64_t b = desc_sw128(smem_u32(smem + st * C::STAGE + C::A_BYTES));
  #pragma unroll
            for (int k = 0; k < BK / 32; ++k)  // 32 bytes of K each: +2 in the descriptors' 16-byte units
              umma_f8(tmem + ab * BN, a + 2 * k, b + 2 * k, idesc, k != 0);
            umma_commit(&empty[st]);
            umma_commit(&acc_full[ab]);
            if (++st == C::STAGES) { st = 0; ph ^= 1; }
            if (++ab == C::NACC) { ab = 0; ap ^= 1; }
          }
        }
      }
    } else {
      // scales, each of the two warps half of a block's: U blocks at a time, so that
      // their loads are in flight together (one block at a time, the loads' latency
      // is the time of a block)
      constexpr int U = C::SU, V = C::SW <= 64 ? 1 : BM / 64, W = TM && BN > BM ? 2 : 1;
      int sr = 0;
      uint32_t sp = 0;
      bool ok = true;
      for (int t = tile0; t < tiles && ok; t += step) {
        const int m = t % args.MT, n = t / args.MT;
        const int t0 = TM ? m * BM : n * bn, wb = TM ? n * bn / BM : m;  // first token, first block of weight rows
        for (int kb = kb0; kb < kb1 && ok; kb += U) {
          float v[U][V], w[U][W];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int k = min(kb + u, kb1 - 1);
#pragma unroll
            for (int i = 0; i < W; ++i)
              w[u][i] = *(args.sw + static_cast<long long>(min(wb + i, (args.N - 1) / BM)) * args.KB + k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int c = (warp - 2) * 32 + lane + 64 * i;
              v[u][i] = t0 + c < args.T && (TM || c < bn) ? *(args.sx + static_cast<long long>(k) * args.T + t0 + c) : 0.0f;
            }
          }
          ok = wait_bar(&s_empty[sr], sp ^ 1, ctl);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int c = (warp - 2) * 32 + lane + 64 * i;
#pragma unroll
              for (int x = 0; x < W; ++x)
                if (TM || c < BN) scales[(sr * U + u) * C::SW + x * BM + c] = v[u][i] * w[u][x];
            }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_full[sr]);
          if (++sr == C::SR) { sr = 0; sp ^= 1; }
        }
      }
    }
  } else {
    if constexpr (C::REGS > 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
    const int quad = warp & 3, group = (warp - EPI_WARP0) >> 2;
    const int row = quad * 32 + lane;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    constexpr int GROUPS = C::EW / 4;
    // column of load i: the column groups take halves of the tile (TM: each within
    // one block of weight rows), or every other load of the columns in use
    auto col = [&](int i) { return TM ? (group * C::CHUNKS + i) * C::CH : (i * GROUPS + group) * C::CH; };
    int ab = 0, sr = 0;
    uint32_t ap = 0, sp = 0;
    bool ok = true;
    for (int t = tile0; t < tiles && ok; t += step) {
      const int r = t % args.MT * BM + row, c = t / args.MT * bn;  // this thread's row, the tile's first column
      unsigned long long acc[C::CHUNKS][C::CH / 2];  // two fp32 each
#pragma unroll
      for (int i = 0; i < C::CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < C::CH / 2; ++j) acc[i][j] = 0ull;
      if constexpr (TM) {
        // the next load is in flight while a load's columns are added, across blocks
        // too: a block's accumulator is given back once its last load has landed
        static_assert(C::CHUNKS % 2 == 0, "two load buffers, each block starts with the first");
        uint32_t d[2][32];
        float sc = 0.0f, sc_next = 0.0f;
        int u = 0;            // block within the scales' hand-over
        bool ready = false;   // the next accumulator was seen complete
        auto begin = [&]() {  // the next block's scale and first load
          if (u == 0) ok = wait_bar(&s_full[sr], sp, ctl);
          if (!ready) ok = ok && wait_bar(&acc_full[ab], ap, ctl);
          ok = __all_sync(0xffffffffu, ok);  // tcgen05.ld is warp-wide
          if (!ok) return;
          sc_next = scales[(sr * C::SU + u) * C::SW + (BN > BM ? group * BM : 0) + row];
          tc_fence_after();
          tmem_issue(tbase + ab * BN + col(0), d[0]);
        };
        begin();
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          sc = sc_next;
#pragma unroll
          for (int i = 0; i < C::CHUNKS; ++i) {
            tmem_wait(d[i & 1]);
            if (i + 1 < C::CHUNKS) {
              tmem_issue(tbase + ab * BN + col(i + 1), d[(i + 1) & 1]);
              if (i + 2 == C::CHUNKS) {
                const bool wrap = ab + 1 == C::NACC;
                ready = mbar_test(&acc_full[wrap ? 0 : ab + 1], wrap ? ap ^ 1 : ap);
              }
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&acc_empty[ab]);
              if (++ab == C::NACC) { ab = 0; ap ^= 1; }
              if (++u == C::SU || kb + 1 == kb1) {
                u = 0;
                if (lane == 0) mbar_arrive(&s_empty[sr]);
                if (++sr == C::SR) { sr = 0; sp ^= 1; }
              }
              if (kb + 1 < kb1) begin();
            }
            add_scaled(acc[i], d[i & 1], sc);
          }
        }
      } else {
        for (int kb = kb0; kb < kb1; ++kb) {
          const int u = (kb - kb0) % C::SU;  // block within the scales' hand-over
          ok = (u > 0 || wait_bar(&s_full[sr], sp, ctl)) && wait_bar(&acc_full[ab], ap, ctl);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const float* s = scales + (sr * C::SU + u) * C::SW;
#pragma unroll
          for (int i = 0; i < C::CHUNKS; ++i) {
            const int c0 = col(i);
            if (c0 >= bn) break;
            uint32_t d[C::CH];
            tmem_read(tbase + ab * BN + c0, d);
#pragma unroll
            for (int j = 0; j < C::CH / 4; ++j) {
              const unsigned long long d0 = static_cast<unsigned long long>(d[4 * j + 1]) << 32 | d[4 * j];
              const unsigned long long d1 = static_cast<unsigned long long>(d[4 * j + 3]) << 32 | d[4 * j + 2];
              const ulonglong2 sc = *reinterpret_cast<const ulonglong2*>(s + c0 + 4 * j);
              asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i][2 * j]) : "l"(d0), "l"(sc.x));
              asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i][2 * j + 1]) : "l"(d1), "l"(sc.y));
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[ab]);
          if (++ab == C::NACC) { ab = 0; ap ^= 1; }
          if (u + 1 == C::SU || kb + 1 == kb1) {
            if (lane == 0) mbar_arrive(&s_empty[sr]);
            if (++sr == C::SR) { sr = 0; sp ^= 1; }
          }
        }
      }
      if (!ok) break;
      float* part = reinterpret_cast<float*>(smem);  // every product of this CTA is complete
#pragma unroll
      for (int i = 0; i < C::CHUNKS; ++i) {
        const int c0 = col(i);
        if (!TM && c0 >= bn) break;
        float v[C::CH];
#pragma unroll
        for (int j = 0; j < C::CH; ++j) v[j] = __uint_as_float(static_cast<uint32_t>(acc[i][j / 2] >> (32 * (j & 1))));
        if (split > 1) {
          if constexpr (TM) {  // token by token
#pragma unroll
            for (int j = 0; j < C::CH; j += 4)
              *reinterpret_cast<float4*>(part + row * C::PITCH + c0 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < C::CH; ++j) part[(c0 + j) * C::PITCH + row] = v[j];
          }
        } else if constexpr (TM) {
          // a lane has a row; rows are stored piece by piece across the lanes, 16, 8 or
          // 4 bytes each as the row length allows (straight from the lanes, every store
          // would touch 32 rows: 581 x 480 x 2698 24.0 us instead of 6.7, 4096 x 4096 x
          // 9216 161 instead of 152)
          uint8_t* place = smem + C::OFF_O + (warp - EPI_WARP0) * C::OUT_PLACE;
          const int r0 = r - lane, n0 = c + c0;  // first row and column of the place
          uint16_t* dst = args.out + static_cast<long long>(r0) * args.N + n0;
          uint32_t w[C::CH / 2];
#pragma unroll
          for (int j = 0; j < C::CH / 2; ++j) w[j] = bf16_pair(v[2 * j], v[2 * j + 1]);
          // with an odd row length every other row begins between two words of memory:
          // its words hold columns 2 j - 1, 2 j, and its first and last column go alone
          const bool odd = args.N % 2 && (static_cast<long long>(r) * args.N + n0) % 2;
          if (odd) {
            uint16_t* own = dst + static_cast<long long>(lane) * args.N;
            if (r < args.T && n0 < args.N) own[0] = static_cast<uint16_t>(w[0]);
            if (r < args.T && n0 + C::CH - 1 < args.N) own[C::CH - 1] = static_cast<uint16_t>(w[C::CH / 2 - 1] >> 16);
#pragma unroll
            for (int j = C::CH / 2 - 1; j > 0; --j) w[j] = __byte_perm(w[j - 1], w[j], 0x5432);
          }
#pragma unroll
          for (int j = 0; j < C::CH / 2; j += 4)
            *reinterpret_cast<uint4*>(place + lane * C::OUT_PITCH + j * 4) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
          __syncwarp();
          auto leave = [&](auto piece) {  // pieces of this many bytes, consecutive lanes along a row
            using V = decltype(piece);
            constexpr int L = 64 / sizeof(V), E = sizeof(V) / 2;
#pragma unroll 8
            for (int x = 0; x < 32; x += 32 / L) {
              const int y = x + lane / L, k = lane % L * E;
              const V u = *reinterpret_cast<const V*>(place + y * C::OUT_PITCH + k * 2);
              if (r0 + y < args.T && n0 + k < args.N) *reinterpret_cast<V*>(dst + static_cast<long long>(y) * args.N + k) = u;
            }
          };
          if (args.N % 8 == 0) {
            leave(uint4());
          } else if (args.N % 4 == 0) {
            leave(uint2());
          } else if (args.N % 2 == 0) {
            leave(uint32_t());
          } else {
            const uint32_t odds = __ballot_sync(0xffffffffu, odd);
#pragma unroll 8
            for (int x = 0; x < 32; x += 2) {
              const int y = x + (lane >> 4), shift = odds >> y & 1, k = (lane & 15) * 2 - shift;
              const uint32_t u = *reinterpret_cast<const uint32_t*>(place + y * C::OUT_PITCH + (lane & 15) * 4);
              uint16_t* to = dst + static_cast<long long>(y) * args.N + k;
              if (r0 + y < args.T && k >= 0) {
                if (n0 + k + 1 < args.N) *reinterpret_cast<uint32_t*>(to) = u;
                else if (n0 + k < args.N) *to = static_cast<uint16_t>(u);
              }
            }
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int j = 0; j < C::CH; ++j)
            if (r < args.N && c0 + j < bn && c + c0 + j < args.T)
              args.out[static_cast<long long>(c + c0 + j) * args.N + r] = f32_to_bf16(v[j]);
        }
      }
    }
  }

  __syncthreads();
  if (split > 1) {
    cluster_sync();  // every CTA's partial sums are written
    if (warp >= EPI_WARP0) {
      const int e = threadIdx.x - EPI_WARP0 * 32;
      if constexpr (TM) {  // a token's columns along the lanes, four each
        constexpr int LANES = BN / 4, ROWS = C::EW * 32 / LANES;
        const int m0 = tile0 % args.MT * BM, n = tile0 / args.MT * bn + e % LANES * 4;
        for (int r = BM * rank / split + e / LANES; r < BM * (rank + 1) / split; r += ROWS) {
          if (m0 + r >= args.T || n >= args.N) continue;
          const uint32_t at = smem_u32(smem) + (r * C::PITCH + e % LANES * 4) * 4;
          float4 v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = x < split ? ld_cluster4(at, x) : make_float4(0.f, 0.f, 0.f, 0.f);
          float4 sum = v[0];
#pragma unroll
          for (int x = 1; x < 8; ++x)
            sum = make_float4(sum.x + v[x].x, sum.y + v[x].y, sum.z + v[x].z, sum.w + v[x].w);
          uint16_t* dst = args.out + static_cast<long long>(m0 + r) * args.N + n;
          if (args.N % 4 == 0) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_pair(sum.x, sum.y), bf16_pair(sum.z, sum.w));
          } else if (args.N % 2 == 0) {
            reinterpret_cast<uint32_t*>(dst)[0] = bf16_pair(sum.x, sum.y);
            if (n + 2 < args.N) reinterpret_cast<uint32_t*>(dst)[1] = bf16_pair(sum.z, sum.w);
          } else {
            const float w[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < args.N) dst[j] = f32_to_bf16(w[j]);
          }
        }
      } else {
        const int row = e & (BM - 1), n = tile0 % args.MT * BM + row, t0 = tile0 / args.MT * bn;
        for (int c = bn * rank / split + (e >> 7); c < bn * (rank + 1) / split; c += C::EW / 4) {
          if (n >= args.N || t0 + c >= args.T) continue;
          const uint32_t at = smem_u32(smem) + (c * C::PITCH + row) * 4;
          float v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = x < split ? ld_cluster(at, x) : 0.0f;
          float sum = v[0];
#pragma unroll
          for (int x = 1; x < 8; ++x) sum += v[x];
          args.out[static_cast<long long>(t0 + c) * args.N + n] = f32_to_bf16(sum);
        }
      }
    }
    __syncthreads();
    cluster_sync();  // no CTA leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
  }
}

// ------------------------------------------------------------------ host side

// Set once per device: the kernel's shared memory, and how many clusters of 2..8
// CTAs the device holds at a time (the SMs of a GPC bound it; a cluster that does
// not fit waits for a whole one to end).
template <bool TM, int BN>
static int clusters(int dev, int split) {
  using C = Cfg<TM, BN>;
  static int n[64][9] = {};
  if (n[dev][0] == 0) {
    if (cudaFuncSetAttribute(fp8_linear_kernel<TM, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return -1;
    for (int x = 2; x <= 8; ++x) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(x);
      cfg.blockDim = dim3(C::THREADS);
      cfg.dynamicSmemBytes = C::SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = x;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n[dev][x], fp8_linear_kernel<TM, BN>, &cfg) != cudaSuccess) return -1;
    }
    n[dev][1] = num_sms() * C::CTAS;
    n[dev][0] = 1;
  }
  return n[dev][split];
}

template <bool TM, int BN>
static int launch(const uint8_t* x8, const uint8_t* w8, int K, Args a, cudaStream_t s) {
  using C = Cfg<TM, BN>;
  int dev = 0;
  SG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || clusters<TM, BN>(dev, 1) < 0) return SG_ERR_CUDA;
  a.MT = ((TM ? a.T : a.N) + BM - 1) / BM;
  a.NT = ((TM ? a.N : a.T) + a.bn - 1) / a.bn;
  if (static_cast<long long>(a.MT) * a.NT > (1 << 27)) return SG_ERR_SHAPE;
  const int tiles = a.MT * a.NT;
  const void* row_op = TM ? x8 : w8;
  const void* col_op = TM ? w8 : x8;
  CUtensorMap ma, mb;
  if (!make_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row_op, K, TM ? a.T : a.N, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, col_op, K, TM ? a.N : a.T, BK, a.bn, CU_TENSOR_MAP_SWIZZLE_128B))
    return SG_ERR_CUDA;
  const int slots = num_sms() * C::CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.split > 1 ? tiles * a.split : tiles < slots ? tiles : slots);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_after_previous
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  SG_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_linear_kernel<TM, BN>, ma, mb, a));
  return SG_OK;
}

}  // namespace f8

int f8_device_status(int reset) {
  int v = 0;
  SG_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_device_status, sizeof(int)));
  if (reset) {
    const int zero = 0;
    SG_CUDA_TRY(cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int)));
  }
  return v;
}

}  // namespace sg

extern "C" int sg_fp8_linear(const uint8_t* x8, const float* x_scales, const uint8_t* w8, const float* w_scales, int T,
                             int K, int N, uint16_t* out, void* stream) {
  using namespace sg::f8;
  if (T < 0) return SG_ERR_INVALID_ARG;
  if (K < 16 || K % 16 || N < 1) return SG_ERR_SHAPE;
  if (T == 0) return SG_OK;
  if (!x8 || !x_scales || !w8 || !w_scales || !out) return SG_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(x8) | reinterpret_cast<uintptr_t>(w8) | reinterpret_cast<uintptr_t>(out)) & 15)
    return SG_ERR_INVALID_ARG;
  Args a = {};
  a.sx = x_scales; a.sw = w_scales; a.out = out;
  a.T = T; a.N = N;
  a.KB = (K + BK - 1) / BK;
  cudaStream_t s = (cudaStream_t)stream;
  if (T <= 64) {
    // The weights' bytes are the cost: as many CTAs as stream them well.  More than
    // five for every three SMs leave clusters waiting for a place (16 x 2048 x 5120,
    // 40 tiles: split 4 7.0 us, 6 6.7, 7 7.5, 8 10.3; 16 x 4096 x 9216, 72 tiles:
    // split 2 13.0 us, 3 12.4, 4 17.2).
    const int tiles = (N + BM - 1) / BM, most = num_sms() * 5 / 3;
    a.split = 1;
    while (a.split < 8 && a.split < a.KB && static_cast<long long>(tiles) * (a.split + 1) <= most) ++a.split;
    a.bn = T <= 16 ? 16 : (T + 15) / 16 * 16;
    if (T <= 16) return launch<false, 16>(x8, w8, K, a, s);
    if (T <= 32) return launch<false, 32>(x8, w8, K, a, s);
    return launch<false, 64>(x8, w8, K, a, s);
  }
  // Tile width and split by a count of time, in 0.1 us: a block of k takes a CTA 4.0
  // (64 columns; 6.0 with two CTAs on an SM), 4.2 (128) or 5.2 (256), joining a
  // split 30, 40 or 60.  (128 x 4096 x 9216: 128 columns split in two 14.7 us, whole
  // 17.5, 64 columns 16.9, 256 split in three 16.5; 333 rows: 256 columns 23.7, 128
  // 31, 64 32; 256 rows: 128 columns 18.2, 64 20.0, 256 25; 128 x 8192 x 1024: 64
  // columns split in eight 10.4, whole 27.)
  const int sms = num_sms();
  int dev = 0;
  SG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return SG_ERR_CUDA;
  const long long rows = (T + BM - 1) / BM;
  double best = 1e30;
  for (int bn = 64; bn <= 256; bn *= 2) {
    const long long tiles = rows * ((N + bn - 1) / bn);
    for (int split = 1; split <= 8 && split <= a.KB; ++split) {
      const long long ctas = tiles * split, slots = bn == 64 ? 2 * sms : sms;
      if (split > 1 && tiles > (bn == 64    ? clusters<true, 64>(dev, split)
                                : bn == 128 ? clusters<true, 128>(dev, split)
                                            : clusters<true, 256>(dev, split)))
        break;
      const double block = bn == 64 ? (ctas > sms ? 6.0 : 4.0) : bn == 128 ? 4.2 : 5.2;
      const double cost = static_cast<double>((ctas + slots - 1) / slots) * ((a.KB + split - 1) / split) * block +
                          (split == 1 ? 0.0 : bn == 64 ? 30.0 : bn == 128 ? 40.0 : 60.0);
      if (cost < best) {
        best = cost;
        a.bn = bn;
        a.split = split;
      }
    }
  }
  if (a.bn == 64) return launch<true, 64>(x8, w8, K, a, s);
  if (a.bn == 128) return launch<true, 128>(x8, w8, K, a, s);
  return launch<true, 256>(x8, w8, K, a, s);
}
