// Grouped NVFP4 expert GEMM on the block-scaled 4-bit path of the
// 5th-generation tensor cores (tcgen05 kind::mxf4nvf4).
//
// Problem: for every expert e and every row r of it
//   D[r, n] = bf16(ga * gb[e] * sum_k (a[r,k] sa[r,k/16]) (b[e,n,k] sb[e,n,k/16]))
// with E2M1 codes a, b (two per byte), E4M3 scales sa, sb for 16 elements
// along K, and float32 global scales ga (activations) and gb[e] (weights).
// The tensor core multiplies code * scale products exactly and sums them in
// fp32; the epilogue applies the global scales in fp32 and rounds once.
// SWIGLU mode computes g and u of 128 output columns, rounds both to bf16,
// applies swiglu_f32, rounds h to bf16 and quantises it (nvfp4.cuh) with the
// output's global scale: bit for bit the plain GEMM, fused_swiglu and
// nvfp4_quantize in a row, without their passes over memory.
//
// Tiling.  The weights are the MMA's M operand (two boxes of 128 rows), the
// tokens its N operand (up to kTok, rounded up to 16): a tile's cost then
// follows its token count, and a weight row passes through shared memory once
// for every chunk of tokens.  An expert's rows are cut into equal chunks of at
// most kTok.  Units are (expert, n-tile, chunk), chunk fastest, so chunks
// that share a weight tile are taken at about the same time by neighbouring
// CTAs and the weight tile comes from HBM once.  A persistent grid of one CTA
// per SM: CTA i starts with unit i and takes its further ones from an atomic
// counter in caller scratch, or with a static stride where there is none.
//
// K runs in stages of 256 elements: one 128-byte swizzled row of codes, four
// MMAs of K=64, and 16 scale bytes a row.  The MMA reads scales from TMEM,
// where a 128-row tile of the four scales of one MMA is 32 lanes x 4 columns
// (row r in lane r % 32, column r / 32), the same in all four lane quarters.
// Four scale warps, one for each quarter, write them there with tcgen05.st: a
// lane takes its 16 bytes of each weight tile from shared memory (the weight
// scales lie in global memory in that order, laid out once, and arrive by bulk
// copies) and the 16 bytes of each of its token rows, plain rows [rows, K/16]
// that start at any expert boundary, from there too where TMA can load them
// (K % 256 == 0: rows of whole 16-byte pieces) and from global memory
// otherwise.  (Loading them from global memory always costs 45 to 70 % more
// time at 128 to 1024 rows an expert: 32 lines a load, in four warps.  So a K
// that is no multiple of 256 costs: N=4096, K=2112 against 2304 takes 39 and 37
// us at 32 experts x 16 rows, 50 and 45 at 32 x 128, 124 and 102 at 16 x 1024.)
// Copying the weights' tiles with tcgen05.cp from the MMA warp instead is 1 to
// 9 % slower (down product, 16 experts of 1024 rows: 171 against 156 us): eight
// more instructions a stage in the lane that paces the MMAs.
//
// Bounds, measured on a B200 with 64 experts, H=7168, I=2048 (6.54 TB/s copy):
// up to 64 rows an expert the weights' stream, gate/up 163 to 167 us = 6.5 to 6.3
// TB/s; at 128 rows 190 us = 5.6 TB/s, where a tile takes both accumulators and
// its epilogue's first part stands between two main loops; at 1024 rows (16
// experts) 239 us = 4.0 PFLOP/s in a burst and 279 us = 3.5 PFLOP/s in a long run,
// where the power cap holds the SM clock at 1492 MHz.  That is 291 stages of 62
// KB for an SM, 0.82 and 0.96 us (1430 cycles) each with the gaps between main
// loops counted in: bound by the loads into shared memory and those gaps.
//
// One CTA = 16 warps:
//   warp 0       takes units; TMA producer of the weights' codes
//   warp 1       MMA issuer: 4 x 2 MMAs a stage
//   warps 2-9    epilogue, two groups of four (warp w reads TMEM lanes
//                32*(w%4)..+31 = its 32 weight rows; the groups alternate
//                chunks of 16 tokens).  A chunk comes out of TMEM as bf16 pairs
//                of the two boxes (g and u, or columns c and c + 128), the next
//                one's load under its arithmetic.  bf16 outputs go straight to
//                memory, 4 bytes a lane after neighbours have traded; for NVFP4 outputs the
//                warp turns its 16 x 32 piece in shared memory, so that a lane
//                holds one block of 16 outputs of a token
//   warps 10-13  scales: shared memory -> TMEM
//   warp 14      TMA producer of the tokens' codes
//   warp 15      TMA producer of scales, into a ring of their own: they are in
//                TMEM by the time the codes land
//
// TMEM: columns 0..383 hold the accumulators (a unit of up to 96 token
// columns takes half of them, so its epilogue overlaps the next unit's main
// loop entirely), 384..511 two buffers of scales (weights 2 boxes x 4 MMAs x 4
// columns, tokens 4 x 8).  A buffer is overwritten only after the MMAs that
// read it have completed (the empty barrier of two stages before).
//
// Waits are bounded as in grouped_gemm.cu.
#include <initializer_list>

#include "nvfp4.cuh"
#include "swiglu.cuh"
#include "umma.cuh"

namespace lsek {
namespace fp4 {

constexpr int kStepK = 64;                        // K of one MMA
constexpr int kSteps = 4;                         // MMAs (per box) of a stage
constexpr int kRowBytes = kSteps * kStepK / 2;    // 128: one swizzle row
constexpr int kBoxRows = 128;                     // weight rows of a box = MMA M
constexpr int kBoxBytes = kBoxRows * kRowBytes;   // 16 KB
constexpr int kSfTile = 512;                      // scales of 128 rows for one MMA
constexpr int kSfBoxBytes = kSteps * kSfTile;     // 2 KB
constexpr int kEpiWarps = 8;
constexpr int kSfWarps = 4;                       // one for each lane quarter of TMEM
constexpr int kFirstSfWarp = 2 + kEpiWarps;
constexpr int kTokWarp = kFirstSfWarp + kSfWarps; // TMA producer of the tokens' codes
constexpr int kSfLoadWarp = kTokWarp + 1;         // TMA producer of scales
constexpr int kThreads = 32 * (kSfLoadWarp + 1);
constexpr int kUnitQ = 4;                         // unit ids in flight between warps
constexpr int kMaxExperts = 1024;
constexpr int kAccCols = 192;                     // TMEM columns of an accumulator slot
constexpr int kSfCol = 2 * kAccCols;              // first column of the scale buffers
constexpr int kSfBufCols = 64;
constexpr int kTmemCols = 512;
constexpr int kStagePitch = 80;                   // epilogue: bytes of a token's 32 bf16 (+ pad)

constexpr int kTok = 192;                         // most token rows of a unit
constexpr int kHalves = 2;                        // 128-row scale tiles of the tokens
constexpr int kRecs = 8;                          // stages in flight at most
constexpr int kSfStages = 3;
constexpr int kSfTokOff = 2 * kSfBoxBytes;        // token scales, 16 bytes a row
constexpr int kSfStageBytes = kSfTokOff + kTok * 16;

// The ring of codes is given out in bytes: a stage takes its two weight boxes
// (16 KB each) and 128 bytes for each token row, so that a decode batch has
// five stages in flight and an expert of 144 rows nearly four.  RING is what
// shared memory leaves beside the unit table of MAX_E experts.
template <int RING, int MAX_E>
struct Geom {
  static constexpr uint32_t kRing = RING;
  static constexpr int kMaxE = MAX_E;
  static_assert(RING % 1024 == 0, "swizzled boxes start on 1 KB");
  static_assert(RING >= 2 * (2 * kBoxBytes + kTok * kRowBytes), "two of the largest stages fit");
};
using GeomFull = Geom<192 * 1024, 256>;
using GeomWide = Geom<184 * 1024, kMaxExperts>;

// Position in the ring.  Every role walks the same stages and keeps its own
// copy; stage j uses record j % kRecs (parity (j / kRecs) & 1).
template <class G>
struct RingPos {
  uint32_t j = 0;    // stages so far
  uint32_t off = 0;  // where the next part goes
  uint32_t w0, w1, tok;  // parts of the current stage
  __device__ __forceinline__ int rec() const { return static_cast<int>(j % kRecs); }
  __device__ __forceinline__ uint32_t parity() const { return (j / kRecs) & 1u; }
  // Lays the next stage out: its boxes of weights and its token rows, each in
  // one piece; a piece that would cross the ring's end starts at 0 instead.
  // Returns the bytes taken, skipped ones included.
  __device__ __forceinline__ uint32_t layout(int boxes, uint32_t tok_bytes) {
    uint32_t span = 0;
    auto place = [&](uint32_t size) -> uint32_t {
      if (off + size > G::kRing) {
        span += G::kRing - off;
        off = 0;
      }
      const uint32_t at = off;
      off += size;
      span += size;
      return at;
    };
    w0 = place(kBoxBytes);
    w1 = boxes == 2 ? place(kBoxBytes) : 0u;
    tok = place(tok_bytes);
    return span;
  }
};

template <class G>
struct SmemT {
  uint8_t ring[G::kRing];  // 1024-byte aligned
  uint8_t sf_ring[kSfStages][kSfStageBytes];
  uint8_t turn[kEpiWarps][16 * kStagePitch];
  uint64_t full_bar[kRecs];
  uint64_t empty_bar[kRecs];
  uint64_t sf_full_bar[kSfStages];
  uint64_t sf_empty_bar[kSfStages];
  uint64_t sf_bar[2];             // a TMEM scale buffer is filled
  uint64_t acc_full_bar[2];
  uint64_t acc_empty_bar[2];
  uint64_t mma_done_bar;
  uint64_t q_full[kUnitQ];
  uint64_t q_empty[kUnitQ];
  int32_t unit_q[kUnitQ];
  uint32_t span[2][kRecs];  // ring bytes of each outstanding stage, for each producer of codes
  uint32_t tmem_base;
  int32_t abort;
  int32_t warp_tot[kThreads / 32];
  int32_t offs[G::kMaxE + 1];
  int32_t cum[G::kMaxE + 1];
};
template <class G>
constexpr size_t smem_bytes() {
  return sizeof(SmemT<G>) + 1024;
}
static_assert(smem_bytes<GeomFull>() <= 227 * 1024, "shared memory budget");
static_assert(smem_bytes<GeomWide>() <= 227 * 1024, "shared memory budget");

struct Params {
  const int32_t* offsets;  // [E+1]
  int num_experts;
  int rows;                // rows of A and of the output
  int steps;               // K / 64
  int n_tiles;             // n-tiles per expert
  int b_rows;              // weight rows per expert
  int b_tile_rows;         // first-box row step per n-tile
  int b_second;            // row offset of the second box
  int sf_tiles;            // 128-row scale tiles per expert
  int sf_tile_step;        // tile step per n-tile of the first box
  int sf_second;           // tile offset of the second box
  const uint8_t* a_sf;     // [rows, K/16]
  const uint8_t* b_sf;     // [E, sf_tiles, steps, 512]
  const float* a_global;   // one value, or null: 1
  const float* b_global;   // [E], or null: 1
  const float* out_global; // SWIGLU: the output's global scale, or null: 1
  __nv_bfloat16* D;        // plain: [rows, n_out]
  uint8_t* out_codes;      // SWIGLU: [rows, n_out/2]
  uint8_t* out_sf;         // SWIGLU: [rows, n_out/16]
  int out_tile_cols;       // output columns per tile
  int n_out;
  float swiglu_limit;
  int32_t* counter;        // zeroed counter of the units past the first of each CTA, or null
  int sf_by_tma;           // rows of a_sf are multiples of 16 bytes (K % 256 == 0)
};

// Tensor maps: weights in boxes of 128 rows; tokens and their scales in boxes of
// 16 << i rows, so that any multiple of 16 up to 192 takes at most four loads
// (each costs its lane about 50 cycles).
struct Maps {
  CUtensorMap b, a[4], s[4];
};

// ---- PTX ----------------------------------------------------------------------

// mbar_wait for chains that have a wait in every link: the first try is inline
// (the call costs hundreds of cycles even on a completed barrier), and later
// ones let the hardware suspend the warp for up to 20 us, so that waiting warps
// leave the issue slots to the epilogue.
__device__ __forceinline__ bool wait_bar_slow(uint64_t* bar, uint32_t parity,
                                              volatile int32_t* abort, int32_t code,
                                              bool honor_abort) {
  const uint64_t t0 = global_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (honor_abort && *abort) return false;
    if (global_ns() - t0 > kWaitLimitNs) {
      *abort = 1;
      report_device_error(code);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int32_t* abort,
                                         int32_t code, bool honor_abort = true) {
  return mbar_try_wait(bar, parity) || wait_bar_slow(bar, parity, abort, code, honor_abort);
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
// Waits for TMEM loads; the registers that they fill are operands, so that no
// use of them can be moved in front.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]),
                 "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]),
                 "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]),
                 "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]),
                 "+r"(b[6]), "+r"(b[7]), "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]),
                 "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void umma_fp4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X"
      " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: A and B E2M1 (1 in bits 7-9 and 10-11), scales E4M3
// (bit 23 = 0), N >> 3 in bits 17-22, M >> 7 in bits 27-28, scale ids 0, K = 64.
__device__ __forceinline__ uint32_t fp4_idesc(int nn) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(nn >> 3) << 17) |
         (static_cast<uint32_t>(kBoxRows >> 7) << 27);
}

// h = bf16(silu(g) u) of 16 tokens (bf16 pairs) of this lane's column, into the
// turning buffer.  The arithmetic of swiglu_f32, silu(g) = g / (1 + 2^(-g
// log2 e)), two tokens an instruction where there is one and with the
// flush-to-zero forms of the exponential and the reciprocal: half its
// instructions, which bound this epilogue.  Results that are bf16 subnormals
// may come out as zeros of the same sign, which quantise to the same codes
// (their quotients are below 2^-17); the others have swiglu_f32's bits.  Tests
// compare the bits of h for every bf16 g from 2^-126 up, of both signs, with up
// values of three exponents, and the codes behind them.
template <bool CLAMP>
__device__ __forceinline__ void swiglu_turn(const uint32_t (&g2)[8], const uint32_t (&u2)[8],
                                            float limit, uint8_t* turn, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 g = unpack2(g2[i], __nv_bfloat16()), u = unpack2(u2[i], __nv_bfloat16());
    if (CLAMP) {
      g = make_float2(clamp_gate(g.x, limit), clamp_gate(g.y, limit));
      u = make_float2(clamp_up(u.x, limit), clamp_up(u.y, limit));
    }
    const float2 t = mul_f32x2(g.x, g.y, -1.4426950408889634f, -1.4426950408889634f);
    float e0, e1, r0, r1;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t.y));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(__fadd_rn(1.0f, e0)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(__fadd_rn(1.0f, e1)));
    const float2 s = mul_f32x2(g.x, g.y, r0, r1);
    const float2 h = mul_f32x2(s.x, s.y, u.x, u.y);
    const uint32_t pair = pack_bf16x2(h.x, h.y);
    uint16_t* dst = reinterpret_cast<uint16_t*>(turn + 2 * i * kStagePitch) + lane;
    dst[0] = static_cast<uint16_t>(pair);
    dst[kStagePitch / 2] = static_cast<uint16_t>(pair >> 16);
  }
}

// ---- work units -----------------------------------------------------------------

template <class S>
__device__ __forceinline__ int chunks_of(const S& s, int e) {
  const int n = s.offs[e + 1] - s.offs[e];
  return n > 0 ? (n + kTok - 1) / kTok : 0;
}

// n-tile n of expert e against `rows` tokens from row0 on.
struct Unit {
  int e, n, row0, rows;
};

// The largest e with cum[e] <= id is the (non-empty) expert that owns the
// unit; its units are ordered (n-tile, chunk), the chunk fastest.  The chunks
// are equal up to the rounding to 16 rows.
template <class S>
__device__ __forceinline__ Unit decode_unit(const S& s, int num_experts, int id) {
  int lo = 0, hi = num_experts - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.cum[mid] <= id) lo = mid;
    else hi = mid - 1;
  }
  Unit u;
  u.e = lo;
  const int local = id - s.cum[lo];
  const int c = chunks_of(s, lo);
  u.n = local / c;
  const int m = local - u.n * c;
  const int n = s.offs[lo + 1] - s.offs[lo];
  const int per = ((n + c - 1) / c + 15) & ~15;
  u.row0 = s.offs[lo] + m * per;
  u.rows = min(per, n - m * per);
  return u;
}

template <bool SWIGLU, class G>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using Smem = SmemT<G>;
  constexpr int kSfTokCols = 4 * kHalves;            // TMEM columns of the tokens' scales of an MMA
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                     ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int E = p.num_experts;

  // ---- unit table: cum[e] = sum over e' < e of chunks(e') * n_tiles -------------
  // Offsets are clamped to [0, rows]; an expert whose end precedes its start has
  // no units, so every stored row stays inside the output.
  for (int i = tid; i <= E; i += kThreads) {
    int v = __ldg(p.offsets + i);
    v = v < 0 ? 0 : (v > p.rows ? p.rows : v);
    s.offs[i] = v;
  }
  if (tid == 0) s.abort = 0;
  __syncthreads();
  {
    const int per = (E + kThreads - 1) / kThreads;
    const int eb = min(E, tid * per);
    const int ee = min(E, eb + per);
    int local = 0;
    for (int e = eb; e < ee; ++e) local += chunks_of(s, e) * p.n_tiles;
    int incl = local;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 31) s.warp_tot[warp] = incl;
    __syncthreads();
    int run = incl - local;
    for (int w = 0; w < warp; ++w) run += s.warp_tot[w];
    for (int e = eb; e < ee; ++e) {
      s.cum[e] = run;
      run += chunks_of(s, e) * p.n_tiles;
    }
    if (eb < E && ee == E) s.cum[E] = run;
  }

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < kRecs; ++i) {
      mbar_init(&s.full_bar[i], 2);  // both producers of codes
      mbar_init(&s.empty_bar[i], 1);
    }
    for (int i = 0; i < kSfStages; ++i) {
      mbar_init(&s.sf_full_bar[i], 1);
      mbar_init(&s.sf_empty_bar[i], kSfWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.sf_bar[i], kSfWarps);
      mbar_init(&s.acc_full_bar[i], 1);
      mbar_init(&s.acc_empty_bar[i], kEpiWarps);
    }
    mbar_init(&s.mma_done_bar, 1);
    for (int i = 0; i < kUnitQ; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1 + kEpiWarps + kSfWarps + 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.b)) : "memory");
    for (int i = 0; i < 4; ++i)
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.a[i])) : "memory");
    for (int i = 0; i < 4 && p.sf_by_tma; ++i)
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.s[i])) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const uint32_t tmem_base = s.tmem_base;
  const int total = s.cum[E];
  const int num_kb = (p.steps + kSteps - 1) / kSteps;
  volatile int32_t* abort = &s.abort;

  // Columns of a unit's tile and whether its second box holds any of them.
  auto cols_of = [&](const Unit& u) { return min(p.out_tile_cols, p.n_out - u.n * p.out_tile_cols); };
  auto boxes_of = [&](const Unit& u) { return SWIGLU || cols_of(u) > kBoxRows ? 2 : 1; };

  // Both producers of codes: waits until a stage of `span` bytes and its record
  // are free; false on abort.  `held` and `j_free` count what this producer has
  // not yet seen released.
  auto reserve = [&](uint32_t* spans, uint32_t j, uint32_t span, uint32_t& j_free,
                     uint32_t& held) -> bool {
    while (j - j_free >= static_cast<uint32_t>(kRecs) || held + span > G::kRing) {
      const uint32_t r = j_free % kRecs;
      if (!wait_bar(&s.empty_bar[r], (j_free / kRecs) & 1u, abort, kDevErrGemmProducerWait)) return false;
      held -= spans[r];
      ++j_free;
    }
    spans[j % kRecs] = span;
    held += span;
    return true;
  };
  // Token rows r, r + 16 << i, ... of a unit in the largest boxes that fit.
  auto box_of = [](int left) { return left >= 128 ? 3 : left >= 64 ? 2 : left >= 32 ? 1 : 0; };

  if (warp == 0) {
    // ===================== units; TMA producer of the weights' codes =====================
    if (elect_one()) {
      // Normal eviction: the other chunks of an expert find the weights in L2.
      const uint64_t policy = policy_evict_normal();
      bool ok = true;
      RingPos<G> pos;
      uint32_t j_free = 0, held = 0;
      int next = blockIdx.x;
      for (uint32_t qn = 0; ok; ++qn) {
        const int qslot = qn % kUnitQ;
        if (!wait_bar(&s.q_empty[qslot], ((qn / kUnitQ) & 1u) ^ 1u, abort, kDevErrGemmProducerWait)) {
          ok = false;
          break;
        }
        const int unit = next < total ? next : -1;
        s.unit_q[qslot] = unit;
        mbar_arrive(&s.q_full[qslot]);
        if (unit < 0) break;
        const Unit u = decode_unit(s, E, unit);
        const int boxes = boxes_of(u);
        const uint32_t tok_bytes = ((u.rows + 15) & ~15) * kRowBytes;
        const int brow = u.e * p.b_rows + u.n * p.b_tile_rows;
        for (int kb = 0; kb < num_kb; ++kb, ++pos.j) {
          // The next unit is asked for a few stages early, so that the answer is
          // there when this one's loads have been issued.
          if (kb == max(0, num_kb - 3))
            next = gridDim.x + (p.counter ? atomicAdd(p.counter, 1) : unit);
          const uint32_t span = pos.layout(boxes, tok_bytes);
          if (!reserve(s.span[0], pos.j, span, j_free, held)) {
            ok = false;
            break;
          }
          uint64_t* full = &s.full_bar[pos.rec()];
          mbar_expect_tx(full, boxes * kBoxBytes);
          tma_load_2d(s.ring + pos.w0, &maps.b, full, kb * kRowBytes, brow, policy);
          if (boxes == 2)
            tma_load_2d(s.ring + pos.w1, &maps.b, full, kb * kRowBytes, brow + p.b_second, policy);
        }
      }
      if (!ok) {  // let every issued load land before the CTA can exit
        for (uint32_t d = j_free; d < pos.j; ++d)
          wait_bar(&s.full_bar[d % kRecs], (d / kRecs) & 1u, abort, kDevErrGemmProducerWait, false);
      }
    }
  } else if (warp == kTokWarp) {
    // ===================== TMA producer of the tokens' codes =====================
    if (elect_one()) {
      const uint64_t policy = policy_evict_last();  // read by every n-tile
      bool ok = true;
      RingPos<G> pos;
      uint32_t j_free = 0, held = 0;
      for (uint32_t qn = 0; ok; ++qn) {
        const int qslot = qn % kUnitQ;
        if (!wait_bar(&s.q_full[qslot], (qn / kUnitQ) & 1u, abort, kDevErrGemmProducerWait)) {
          ok = false;
          break;
        }
        const int unit = s.unit_q[qslot];
        mbar_arrive(&s.q_empty[qslot]);
        if (unit < 0) break;
        const Unit u = decode_unit(s, E, unit);
        const int nn = (u.rows + 15) & ~15;
        const int boxes = boxes_of(u);
        for (int kb = 0; kb < num_kb; ++kb, ++pos.j) {
          const uint32_t span = pos.layout(boxes, nn * kRowBytes);
          if (!reserve(s.span[1], pos.j, span, j_free, held)) {
            ok = false;
            break;
          }
          uint64_t* full = &s.full_bar[pos.rec()];
          mbar_expect_tx(full, nn * kRowBytes);
          for (int r = 0; r < nn;) {
            const int i = box_of(nn - r);
            tma_load_2d(s.ring + pos.tok + r * kRowBytes, &maps.a[i], full, kb * kRowBytes,
                        u.row0 + r, policy);
            r += 16 << i;
          }
        }
      }
      if (!ok) {
        for (uint32_t d = j_free; d < pos.j; ++d)
          wait_bar(&s.full_bar[d % kRecs], (d / kRecs) & 1u, abort, kDevErrGemmProducerWait, false);
      }
    }
  } else if (warp == kSfLoadWarp) {
    // ===================== TMA producer of scales =====================
    // Runs up to kSfStages stages ahead of the scale warps, so that scales wait in
    // TMEM before their codes land.
    if (elect_one()) {
      const uint64_t policy = policy_evict_last();
      bool ok = true;
      uint32_t j = 0;
      for (uint32_t qn = 0; ok; ++qn) {
        const int qslot = qn % kUnitQ;
        if (!wait_bar(&s.q_full[qslot], (qn / kUnitQ) & 1u, abort, kDevErrGemmScaleWait)) {
          ok = false;
          break;
        }
        const int unit = s.unit_q[qslot];
        mbar_arrive(&s.q_empty[qslot]);
        if (unit < 0) break;
        const Unit u = decode_unit(s, E, unit);
        const int nn = (u.rows + 15) & ~15;
        const int boxes = boxes_of(u);
        const uint8_t* sf = p.b_sf + static_cast<int64_t>(u.e * p.sf_tiles + u.n * p.sf_tile_step) *
                                         p.steps * kSfTile;
        const uint8_t* sf2 = sf + static_cast<int64_t>(p.sf_second) * p.steps * kSfTile;
        for (int kb = 0; kb < num_kb; ++kb, ++j) {
          const uint32_t slot = j % kSfStages;
          if (!wait_bar(&s.sf_empty_bar[slot], ((j / kSfStages) & 1u) ^ 1u, abort, kDevErrGemmScaleWait)) {
            ok = false;
            break;
          }
          uint8_t* st = s.sf_ring[slot];
          uint64_t* full = &s.sf_full_bar[slot];
          const uint32_t bytes = min(kSteps, p.steps - kb * kSteps) * kSfTile;
          mbar_expect_tx(full, boxes * bytes + (p.sf_by_tma ? nn * 16 : 0));
          bulk_load(st, sf, bytes, full);
          if (boxes == 2) bulk_load(st + kSfBoxBytes, sf2, bytes, full);
          sf += kSfBoxBytes;  // a tile has 8 K bytes, more than an int in a long row
          sf2 += kSfBoxBytes;
          if (p.sf_by_tma) {
            for (int r = 0; r < nn;) {
              const int i = box_of(nn - r);
              tma_load_2d(st + kSfTokOff + r * 16, &maps.s[i], full, kb * 16, u.row0 + r, policy);
              r += 16 << i;
            }
          }
        }
      }
      if (!ok) {
        for (uint32_t d = j > kSfStages ? j - kSfStages : 0; d < j; ++d)
          wait_bar(&s.sf_full_bar[d % kSfStages], (d / kSfStages) & 1u, abort, kDevErrGemmScaleWait, false);
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    if (elect_one()) {
      uint32_t ac = 0;  // accumulator slots taken so far
      RingPos<G> pos;
      const uint32_t ring = smem_u32(s.ring);
      bool ok = true;
      for (uint32_t qn = 0; ok; ++qn) {
        const int qslot = qn % kUnitQ;
        if (!wait_bar(&s.q_full[qslot], (qn / kUnitQ) & 1u, abort, kDevErrGemmMmaWait)) break;
        const int unit = s.unit_q[qslot];
        mbar_arrive(&s.q_empty[qslot]);
        if (unit < 0) break;
        const Unit u = decode_unit(s, E, unit);
        const int nn = (u.rows + 15) & ~15;
        const int boxes = boxes_of(u);
        const uint32_t idesc = fp4_idesc(nn);
        const bool two = nn > kAccCols / 2;  // the unit takes both slots
        const uint32_t acc0 = ac & 1u, acc1 = (ac + 1) & 1u;
        if (!wait_bar(&s.acc_empty_bar[acc0], ((ac >> 1) & 1u) ^ 1u, abort, kDevErrGemmMmaWait) ||
            (two && !wait_bar(&s.acc_empty_bar[acc1], (((ac + 1) >> 1) & 1u) ^ 1u, abort,
                              kDevErrGemmMmaWait))) {
          ok = false;
          break;
        }
        ac += two ? 2u : 1u;
        tc_fence_after();
        const uint32_t d0 = tmem_base + (two ? 0u : acc0 * kAccCols);
        const uint32_t d1 = d0 + (two ? kAccCols : kAccCols / 2);
        for (int kb = 0; kb < num_kb; ++kb, ++pos.j) {
          const int rec = pos.rec();
          const uint32_t j = pos.j;
          pos.layout(boxes, nn * kRowBytes);
          if (!wait_bar(&s.full_bar[rec], pos.parity(), abort, kDevErrGemmMmaWait) ||
              !wait_bar(&s.sf_bar[j & 1u], (j >> 1) & 1u, abort, kDevErrGemmMmaWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfb = tmem_base + kSfCol + (j & 1u) * kSfBufCols;  // weights
          const uint32_t sft = sfb + 2 * kSteps * 4;                        // tokens
          const int steps = min(kSteps, p.steps - kb * kSteps);
          for (int k = 0; k < steps; ++k) {
            const uint64_t tok = smem_desc_sw128(ring + pos.tok + k * 32);
            const uint32_t acc_in = (kb | k) != 0 ? 1u : 0u;
            umma_fp4(d0, smem_desc_sw128(ring + pos.w0 + k * 32), tok, idesc, sfb + k * 8,
                     sft + k * kSfTokCols, acc_in);
            if (boxes == 2)
              umma_fp4(d1, smem_desc_sw128(ring + pos.w1 + k * 32), tok, idesc, sfb + k * 8 + 4,
                       sft + k * kSfTokCols, acc_in);
          }
          umma_commit(&s.empty_bar[rec]);
        }
        if (ok) {
          umma_commit(&s.acc_full_bar[acc0]);
          if (two) umma_commit(&s.acc_full_bar[acc1]);
        }
      }
      // Outstanding MMAs read shared memory and write TMEM: finish them first.
      umma_commit(&s.mma_done_bar);
      wait_bar(&s.mma_done_bar, 0, abort, kDevErrGemmMmaWait, false);
    }
  } else if (warp >= kFirstSfWarp && warp < kTokWarp) {
    // ===================== scales (warps 10..13) =====================
    const uint32_t quarter = static_cast<uint32_t>((warp & 3) * 32) << 16;  // its TMEM lanes
    const int sf_row = p.steps * 4;  // scale bytes of a token row
    uint32_t j = 0;
    bool ok = true;
    for (uint32_t qn = 0; ok; ++qn) {
      const int qslot = qn % kUnitQ;
      ok = __all_sync(0xffffffffu, wait_bar(&s.q_full[qslot], (qn / kUnitQ) & 1u, abort,
                                             kDevErrGemmScaleWait));
      if (!ok) break;
      const int unit = s.unit_q[qslot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_empty[qslot]);
      if (unit < 0) break;
      const Unit u = decode_unit(s, E, unit);
      // Without TMA: the scales of stage kb of token row 32 q + lane, word k
      // for MMA k.  Rows past the unit and MMAs past K get zeros.
      auto load_tok = [&](int kb, uint32_t (&t)[4 * kHalves][kSteps]) {
#pragma unroll
        for (int q = 0; q < 4 * kHalves; ++q) {
          const int r = q * 32 + lane;
          const uint8_t* src = p.a_sf + static_cast<int64_t>(u.row0 + r) * sf_row + kb * (4 * kSteps);
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
            t[q][k] = r < u.rows && kb * kSteps + k < p.steps
                          ? __ldg(reinterpret_cast<const uint32_t*>(src) + k)
                          : 0u;
        }
      };
      uint32_t tok[4 * kHalves][kSteps];
      for (int kb = 0; kb < num_kb; ++kb, ++j) {
        const uint32_t slot = j % kSfStages;
        if (!p.sf_by_tma) load_tok(kb, tok);
        ok = __all_sync(0xffffffffu, wait_bar(&s.sf_full_bar[slot], (j / kSfStages) & 1u, abort,
                                               kDevErrGemmScaleWait));
        if (!ok) break;
        const uint8_t* image = s.sf_ring[slot] + lane * 16;
        uint32_t w[2 * kSteps * 4];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint4 v = *reinterpret_cast<const uint4*>(image + b * kSfBoxBytes + k * kSfTile);
            w[(2 * k + b) * 4] = v.x;
            w[(2 * k + b) * 4 + 1] = v.y;
            w[(2 * k + b) * 4 + 2] = v.z;
            w[(2 * k + b) * 4 + 3] = v.w;
          }
        if (p.sf_by_tma) {
#pragma unroll
          for (int q = 0; q < 4 * kHalves; ++q)
            if (q * 32 < kTok) {
              const uint4 v = *reinterpret_cast<const uint4*>(image + kSfTokOff + q * 512);
              tok[q][0] = v.x;
              tok[q][1] = v.y;
              tok[q][2] = v.z;
              tok[q][3] = v.w;
            }
        }
        uint32_t t[kSteps * kSfTokCols];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int q = 0; q < 4 * kHalves; ++q)
            t[k * kSfTokCols + q] = q * 32 < kTok ? tok[q][k] : 0u;
        // The MMAs of two stages before, which read this buffer, have completed.
        if (j >= 2)
          ok = __all_sync(0xffffffffu, wait_bar(&s.empty_bar[(j - 2) % kRecs], ((j - 2) / kRecs) & 1u,
                                                 abort, kDevErrGemmScaleWait));
        if (!ok) break;
        tc_fence_after();
        const uint32_t col = tmem_base + quarter + kSfCol + (j & 1u) * kSfBufCols;
        tmem_st32(col, w);
        tmem_st32(col + 2 * kSteps * 4, t);
        tmem_st_wait();
        tc_fence_before();
        // The slot goes back only now that its bytes have gone through registers to
        // TMEM, and with a proxy fence: these were ordinary loads, and the next
        // bytes come through the async proxy, which overtakes a load that is still
        // under way (a release right after the loads gave 1 % wrong outputs).
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.sf_bar[j & 1u]);
          mbar_arrive(&s.sf_empty_bar[slot]);
        }
      }
    }
  } else {
    // ===================== epilogue (warps 2..9) =====================
    const int q = warp & 3;           // TMEM lane quarter this warp may access
    const int grp = (warp - 2) >> 2;  // chunks of 16 tokens this warp drains: grp, grp + 2, ...
    uint8_t* turn = s.turn[warp - 2];
    const float ga = p.a_global ? __ldg(p.a_global) : 1.0f;
    const float go = SWIGLU && p.out_global ? __ldg(p.out_global) : 1.0f;
    const float six_go = __fmul_rn(6.0f, go);
    uint32_t ac = 0;
    for (uint32_t qn = 0;; ++qn) {
      const int qslot = qn % kUnitQ;
      if (!__all_sync(0xffffffffu, wait_bar(&s.q_full[qslot], (qn / kUnitQ) & 1u, abort,
                                             kDevErrGemmEpilogueWait)))
        break;
      const int unit = s.unit_q[qslot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.q_empty[qslot]);
      if (unit < 0) break;
      const Unit u = decode_unit(s, E, unit);
      const int nn = (u.rows + 15) & ~15;
      const bool two = nn > kAccCols / 2;
      const uint32_t acc0 = ac & 1u, acc1 = (ac + 1) & 1u;
      bool got = wait_bar(&s.acc_full_bar[acc0], (ac >> 1) & 1u, abort, kDevErrGemmEpilogueWait);
      if (two)
        got = wait_bar(&s.acc_full_bar[acc1], ((ac + 1) >> 1) & 1u, abort, kDevErrGemmEpilogueWait) && got;
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      const uint32_t d0 = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                          (two ? 0u : acc0 * kAccCols);
      const uint32_t d1 = d0 + (two ? kAccCols : kAccCols / 2);
      const float alpha = p.b_global ? __fmul_rn(ga, __ldg(p.b_global + u.e)) : ga;
      const int col0 = u.n * p.out_tile_cols;
      const int cols = cols_of(u);
      const int boxes = boxes_of(u);
      const int tok = lane >> 1;                  // after the turn: token and
      const int feat = q * 32 + (lane & 1) * 16;  // first of 16 output columns of the box
      const uint4* mine = reinterpret_cast<const uint4*>(turn + tok * kStagePitch + (lane & 1) * 32);
      auto give_back = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.acc_empty_bar[acc0]);
          if (two) mbar_arrive(&s.acc_empty_bar[acc1]);
        }
      };
      // Chunks of 16 tokens.  A chunk's accumulators are scaled and rounded to
      // bf16 pairs of tokens; then the next chunk's TMEM loads start (or the
      // accumulator goes back) and run under this one's arithmetic.
      uint32_t v0[16], v1[16], p0[8], p1[8];
      auto load_chunk = [&](int t0) {
        tmem_ld16(d0 + t0, v0);
        tmem_ld16(d1 + t0, v1);  // not written by a unit with one box; not used then
      };
      if (grp * 16 < nn) load_chunk(grp * 16);
      const int64_t row0 = u.row0 + grp * 16;
      // SWIGLU: this lane's block of token row0 + tok; else its two columns of the
      // first or second row of a pair
      int64_t at = SWIGLU ? ((row0 + tok) * p.n_out + col0 + feat) / kFp4Block
                          : (row0 + (lane & 1)) * p.n_out + col0 + q * 32 + (lane & ~1);
      const uint32_t trade = (lane & 1) == 0 ? 0x5410u : 0x3276u;
      const int64_t pair_step = 2ll * p.n_out;
      const int64_t at_step = SWIGLU ? 2ll * p.n_out : 32ll * p.n_out;  // 32 rows on
      const bool in0 = (SWIGLU ? feat : q * 32 + lane) < cols, in1 = kBoxRows + q * 32 + lane < cols;
#pragma unroll 1
      for (int t0 = grp * 16; t0 < nn; t0 += 32, at += at_step) {
        tmem_ld_wait(v0, v1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 a = mul_f32x2(__uint_as_float(v0[2 * i]), __uint_as_float(v0[2 * i + 1]), alpha, alpha);
          const float2 b = mul_f32x2(__uint_as_float(v1[2 * i]), __uint_as_float(v1[2 * i + 1]), alpha, alpha);
          p0[i] = pack_bf16x2(a.x, a.y);
          p1[i] = pack_bf16x2(b.x, b.y);
        }
        if (t0 + 32 < nn) load_chunk(t0 + 32);
        else give_back();
        if (SWIGLU) {
          if (p.swiglu_limit > 0.0f) swiglu_turn<true>(p0, p1, p.swiglu_limit, turn, lane);
          else swiglu_turn<false>(p0, p1, 0.0f, turn, lane);
          __syncwarp();
          const uint4 lo = mine[0], hi = mine[1];
          __syncwarp();
          if (t0 + tok < u.rows && in0) {
            const Fp4Block blk = fp4_quantize16<__nv_bfloat16>(lo, hi, go, six_go);
            reinterpret_cast<uint2*>(p.out_codes)[at] = blk.codes;
            p.out_sf[at] = static_cast<uint8_t>(blk.scale);
          }
        } else {
          // Neighbouring lanes trade, so that an even lane has two columns of the
          // even token of a pair and an odd lane those of the odd one.
          __nv_bfloat16* dst = p.D + at;
#pragma unroll
          for (int i = 0; i < 8; ++i, dst += pair_step) {
            const uint32_t o0 = __shfl_xor_sync(0xffffffffu, p0[i], 1);
            const uint32_t o1 = __shfl_xor_sync(0xffffffffu, p1[i], 1);
            if (t0 + 2 * i + (lane & 1) < u.rows) {
              if (in0) *reinterpret_cast<uint32_t*>(dst) = __byte_perm(p0[i], o0, trade);
              if (in1) *reinterpret_cast<uint32_t*>(dst + kBoxRows) = __byte_perm(p1[i], o1, trade);
            }
          }
        }
      }
      if (grp * 16 >= nn) give_back();
      ac += two ? 2u : 1u;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// ---- host side -----------------------------------------------------------------

// 2-D byte map over a [outer, inner] row-major tensor, box [box_rows,
// box_bytes], 128-byte swizzle for boxes of codes (128 bytes wide) and none for
// scales (16 bytes), zero fill out of bounds (code 0 = value 0).
lsek_status make_map(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                     uint32_t box_rows, uint32_t box_bytes = kRowBytes) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (fn == nullptr) return fail(LSEK_ERR_CUDA, "grouped_gemm_nvfp4: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {inner};
  const cuuint32_t box[2] = {box_bytes, box_rows};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims,
                        strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_bytes == kRowBytes ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(LSEK_ERR_CUDA, "grouped_gemm_nvfp4: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return LSEK_OK;
}

template <bool SWIGLU, class G>
lsek_status launch_geom(Params p, const void* A, const void* B, int K, bool zero_counter,
                        cudaStream_t st) {
  static PerDeviceOnce attrs;
  const cudaError_t ae = once_per_device(attrs, [] {
    return cudaFuncSetAttribute(fp4_gemm_kernel<SWIGLU, G>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem_bytes<G>()));
  });
  if (ae != cudaSuccess) return fail(LSEK_ERR_CUDA, "grouped_gemm_nvfp4: %s", cudaGetErrorString(ae));
  Maps m{};
  const uint64_t row_bytes = static_cast<uint64_t>(K) / 2;
  lsek_status s = make_map(&m.b, B, row_bytes, static_cast<uint64_t>(p.num_experts) * p.b_rows,
                           static_cast<uint32_t>(kBoxRows));
  for (int i = 0; i < 4 && s == LSEK_OK; ++i) {
    s = make_map(&m.a[i], A, row_bytes, static_cast<uint64_t>(p.rows), 16u << i);
    if (s == LSEK_OK && p.sf_by_tma)
      s = make_map(&m.s[i], p.a_sf, row_bytes / 8, static_cast<uint64_t>(p.rows), 16u << i, 16u);
  }
  if (s != LSEK_OK) return s;
  // At most rows / kTok full chunks and one partial chunk per non-empty expert.
  const int64_t experts = p.num_experts < p.rows ? p.num_experts : p.rows;
  const int64_t max_units = (p.rows / kTok + experts) * static_cast<int64_t>(p.n_tiles);
  const int grid = static_cast<int>(max_units < num_sms() ? max_units : num_sms());
  // A static stride does without the memset (2 us): where every CTA has one unit
  // at most, and where no expert has more than kTok rows, so that the units are
  // alike (each streams one weight tile; 224 of them: 22.6 against 16.8 us).
  if (max_units <= grid || p.rows <= kTok) p.counter = nullptr;
  if (p.counter != nullptr && zero_counter)
    LSEK_CUDA_TRY(cudaMemsetAsync(p.counter, 0, sizeof(int32_t), st));
  fp4_gemm_kernel<SWIGLU, G><<<grid, kThreads, smem_bytes<G>(), st>>>(m, p);
  return check_launch(SWIGLU ? "grouped_gemm_swiglu_nvfp4" : "grouped_gemm_nvfp4");
}

}  // namespace fp4

lsek_status fp4_take_device_error(int32_t* code) {
  int32_t zero = 0;
  LSEK_CUDA_TRY(cudaMemcpyFromSymbol(code, g_device_error, sizeof(int32_t)));
  LSEK_CUDA_TRY(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int32_t)));
  return LSEK_OK;
}

// Both products; D for the plain one, h_codes / h_scales for gate/up + SwiGLU
// (n_out = I there).  Every argument has been checked.  counter: an int32 of
// device scratch, or null; zero_counter: it has to be zeroed here.
lsek_status grouped_gemm_fp4(bool swiglu, void* D, void* h_codes, void* h_scales, const void* A,
                             const void* a_scales, const void* B, const void* b_tiles,
                             const int32_t* offsets, const float* a_global, const float* b_global,
                             const float* out_global, int E, int rows, int n_out, int K,
                             float limit, int32_t* counter, bool zero_counter, cudaStream_t st) {
  using namespace fp4;
  if (rows == 0 || n_out == 0) return LSEK_OK;
  Params p{};
  p.offsets = offsets;
  p.num_experts = E;
  p.rows = rows;
  p.steps = K / kStepK;
  p.a_sf = static_cast<const uint8_t*>(a_scales);
  p.b_sf = static_cast<const uint8_t*>(b_tiles);
  p.a_global = a_global;
  p.b_global = b_global;
  p.out_global = out_global;
  p.D = static_cast<__nv_bfloat16*>(D);
  p.out_codes = static_cast<uint8_t*>(h_codes);
  p.out_sf = static_cast<uint8_t*>(h_scales);
  p.n_out = n_out;
  p.swiglu_limit = limit;
  p.counter = counter;
  p.sf_by_tma = K % (kSteps * kStepK) == 0 && reinterpret_cast<uintptr_t>(a_scales) % 16 == 0;
  const int col_tiles = static_cast<int>(ceil_div(n_out, kBoxRows));
  if (swiglu) {  // gate rows and up rows are tiled apart
    p.b_rows = 2 * n_out;
    p.b_tile_rows = kBoxRows;
    p.b_second = n_out;
    p.sf_tiles = 2 * col_tiles;
    p.sf_tile_step = 1;
    p.sf_second = col_tiles;
    p.out_tile_cols = kBoxRows;
  } else {
    p.b_rows = n_out;
    p.b_tile_rows = 2 * kBoxRows;
    p.b_second = kBoxRows;
    p.sf_tiles = col_tiles;
    p.sf_tile_step = 2;
    p.sf_second = 1;
    p.out_tile_cols = 2 * kBoxRows;
  }
  p.n_tiles = static_cast<int>(ceil_div(n_out, p.out_tile_cols));
  if (E <= GeomFull::kMaxE)
    return swiglu ? launch_geom<true, GeomFull>(p, A, B, K, zero_counter, st)
                  : launch_geom<false, GeomFull>(p, A, B, K, zero_counter, st);
  return swiglu ? launch_geom<true, GeomWide>(p, A, B, K, zero_counter, st)
                : launch_geom<false, GeomWide>(p, A, B, K, zero_counter, st);
}

namespace {

lsek_status check_fp4_gemm(const char* name, int E, int rows, int n_out, int n_weights, int K,
                           std::initializer_list<const void*> sixteen, const void* a_scales,
                           const int32_t* offsets, const void* workspace) {
  LSEK_REQUIRE(E >= 1, "%s: num_experts must be >= 1", name);
  LSEK_REQUIRE(rows >= 0 && n_out >= 0 && K >= 0, "%s: sizes must be >= 0", name);
  if (E > fp4::kMaxExperts)
    return fail(LSEK_ERR_UNSUPPORTED, "%s: num_experts must be <= %d", name, fp4::kMaxExperts);
  LSEK_REQUIRE(K % fp4::kStepK == 0, "%s: K must be a multiple of %d, got %d", name, fp4::kStepK, K);
  LSEK_REQUIRE(n_out % 32 == 0, "%s: output width must be a multiple of 32, got %d", name, n_out);
  LSEK_REQUIRE(static_cast<int64_t>(E) * n_weights < (1ll << 31),
               "%s: num_experts * weight rows must fit in int32", name);
  if (rows == 0 || n_out == 0) return LSEK_OK;
  LSEK_REQUIRE(K > 0, "%s: K must be > 0 when there are rows to compute", name);
  LSEK_REQUIRE(offsets != nullptr, "%s: expert_offsets is NULL", name);
  // Rows of scales are a multiple of 4 bytes, so that a slice of rows is aligned to that.
  LSEK_REQUIRE(a_scales != nullptr, "%s: NULL tensor pointer", name);
  LSEK_REQUIRE(reinterpret_cast<uintptr_t>(a_scales) % 4 == 0, "%s: a_scales must be 4-byte aligned", name);
  for (const void* t : sixteen) {
    LSEK_REQUIRE(t != nullptr, "%s: NULL tensor pointer", name);
    LSEK_REQUIRE(reinterpret_cast<uintptr_t>(t) % 16 == 0, "%s: tensors must be 16-byte aligned", name);
  }
  LSEK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "%s: workspace must be 4-byte aligned", name);
  return LSEK_OK;
}

int32_t* counter_in(void* workspace, size_t workspace_bytes) {
  return workspace != nullptr && workspace_bytes >= sizeof(int32_t) ? static_cast<int32_t*>(workspace)
                                                                    : nullptr;
}

}  // namespace
}  // namespace lsek

extern "C" lsek_status lsek_grouped_gemm_nvfp4(void* D, const void* A, const void* a_scales,
                                               const void* B, const void* b_scale_tiles,
                                               const int32_t* expert_offsets,
                                               const float* a_global_scale,
                                               const float* b_global_scale, int32_t num_experts,
                                               int32_t rows, int32_t N, int32_t K, void* workspace,
                                               size_t workspace_bytes, void* stream) {
  using namespace lsek;
  const lsek_status s = check_fp4_gemm("grouped_gemm_nvfp4", num_experts, rows, N, N, K,
                                       {D, A, B, b_scale_tiles}, a_scales, expert_offsets, workspace);
  if (s != LSEK_OK) return s;
  return grouped_gemm_fp4(false, D, nullptr, nullptr, A, a_scales, B, b_scale_tiles, expert_offsets,
                          a_global_scale, b_global_scale, nullptr, num_experts, rows, N, K, 0.0f,
                          counter_in(workspace, workspace_bytes), true, static_cast<cudaStream_t>(stream));
}

extern "C" lsek_status lsek_grouped_gemm_swiglu_nvfp4(
    void* h_codes, void* h_scales, const void* A, const void* a_scales, const void* W_gu,
    const void* gu_scale_tiles, const int32_t* expert_offsets, const float* a_global_scale,
    const float* gu_global_scale, const float* h_global_scale, int32_t num_experts, int32_t rows,
    int32_t I, int32_t K, float swiglu_limit, void* workspace, size_t workspace_bytes,
    void* stream) {
  using namespace lsek;
  LSEK_REQUIRE(I >= 0 && I < (1 << 30), "grouped_gemm_swiglu_nvfp4: I out of range");
  const lsek_status s =
      check_fp4_gemm("grouped_gemm_swiglu_nvfp4", num_experts, rows, I, 2 * I, K,
                     {h_codes, h_scales, A, W_gu, gu_scale_tiles}, a_scales, expert_offsets,
                     workspace);
  if (s != LSEK_OK) return s;
  LSEK_REQUIRE(swiglu_limit >= 0.0f, "grouped_gemm_swiglu_nvfp4: swiglu_limit must be >= 0");
  return grouped_gemm_fp4(true, nullptr, h_codes, h_scales, A, a_scales, W_gu, gu_scale_tiles,
                          expert_offsets, a_global_scale, gu_global_scale, h_global_scale,
                          num_experts, rows, I, K, swiglu_limit, counter_in(workspace, workspace_bytes), true,
                          static_cast<cudaStream_t>(stream));
}
