// Ragged attention over a paged or contiguous KV cache on the 5th-generation tensor cores (tcgen05 + TMEM +
// TMA): items of two 128-row MMA tiles (see spf_ragged.cuh for items, units and how the line of units is cut).
//
// One persistent CTA per SM.  The two tiles of an item ("stream A / B": consecutive tokens x the heads of one KV
// head) share every K/V unit of 128 keys.
//
//   warp 0      producer: walks the CTA's parts of items and announces each to the other warps through shared memory;
//               loads its Q tiles, then K and V units through a K ring and a V ring by TMA; a unit of
//               pages smaller than 128 tokens is one copy per page and 64 columns, issued by as many lanes, and a
//               page that is not there is a copy from behind the pool, which fills zeros
//   warps 1, 2  MMA issuers of the streams: S = Q K^T and O += P V (P from TMEM); the steps of the two leave in turn
//               (a token goes back and forth), so that one stream's softmax runs under the other's products
//   warp 3      rows of V units at the edges that no query of the item sees are set to zero before the unit is used: what lies
//               behind the sequence, between the sinks and the window, or in the future may hold NaN, and 0 * NaN
//               would reach the output (scores of such keys are replaced, so K needs no such care)
//   warps 4-7, 8-11  softmax of stream A, B: a thread owns a row; base-2 softmax in fp32 against a reference
//               point that is fixed by the first unit in which the row sees a key and moved only when a unit's
//               sum overflows its limit; P rounded to the inputs' type; the epilogue writes the row.  What describes
//               the item stays in shared memory: the 128 scores of a row leave few registers
//
// The rings, S and P run on across items; Q is loaded as soon as the previous item's last Q K^T is done.
// Every wait is bounded (spf_tc5.cuh).
#include "spf_ragged.cuh"
#include "spf_tc5.cuh"

namespace spf {

constexpr int RT_THREADS = 384, RT_CTAS = 148, RT_UNIT = 128, RT_ROWS = 128;
constexpr int RT_REGS_CONTROL = 104, RT_REGS_SOFTMAX = 200;
static_assert(4 * RT_REGS_CONTROL + 8 * RT_REGS_SOFTMAX <= 12 * 168, "setmaxnreg targets exceed the CTA's register pool");
constexpr uint32_t RT_SLAB = 128 * 128;              // [128 rows][64 elements]
constexpr uint32_t RT_CTRL = 2048;
constexpr int RT_ABSENT = 16;                        // units whose absent pages are remembered

// A part of an item as the producer announces it.  Unit u starts at key key_a + 128 u for u < units_a, at
// key_b + 128 (u - units_a) behind that.
struct alignas(16) RtPart {
  int units, units_a, key_a, key_b;           // units 0: no more parts
  int both, whole, slot, n_tok;               // stream B has rows; the item is whole, else its partial slot
  int heads, pos0, keys, low;                 // keys in [low, keys) or below sinks are seen by some row
  int embed, sink_keys, sink_units, pad;      // unit 0: columns below embed are keys from 0 on; the first sink_units units
                                              // are sinks: of both count the keys below sink_keys
  long long out;                              // offset of the item's first token and head in the output
  // some rows of V unit u must become zeros
  __device__ bool edge(int u) const {
    const int key = key0(u);
    return key < low || key + 128 > keys;
  }
  __device__ int key0(int u) const { return u < units_a ? key_a + u * 128 : key_b + (u - units_a) * 128; }
};
constexpr int RT_PARTS = 2;                          // announced parts

template <int D>
struct RtCfg {
  static constexpr int SLABS = D / 64, KSTEPS = D / 16;
  static constexpr uint32_t TILE = RT_SLAB * SLABS;
  static constexpr int KST = D == 128 ? 3 : 6, VST = D == 128 ? 2 : 5;
  // Pairs of exponentials out of eight that go to the FMA pipe.  At D = 128 the products take as long as the exponentials and
  // none need go there: the last 2K chunk of a 34K prompt with 0 / 1 / 2 of them takes 1022 / 1028 / 1230 us (2 spills), the
  // windowed 32K prompt 1172 / 1190 / 1390.  At D = 64, 0 / 1 / 2 / 3: 779 / 735 / 738 / 783 and 935 / 929 / 967 / 1006 us.
  static constexpr int POLY = D == 128 ? 0 : 1;
  static constexpr bool P_BESIDE = D == 64;        // columns 384 .. 511 are free
  // barriers
  static constexpr int B_PFULL = 0, B_PEMPTY = B_PFULL + RT_PARTS, B_QFULL = B_PEMPTY + RT_PARTS, B_QEMPTY = B_QFULL + 2,
                       B_KFULL = B_QEMPTY + 2, B_KEMPTY = B_KFULL + KST, B_VFULL = B_KEMPTY + KST,
                       B_VEDGE = B_VFULL + VST, B_VEMPTY = B_VEDGE + VST, B_SFULL = B_VEMPTY + VST, B_PREADY = B_SFULL + 2,
                       B_ODONE = B_PREADY + 2, B_TOKEN = B_ODONE + 2, B_N = B_TOKEN + 2;
  static constexpr uint32_t O_TMEM = B_N * 8, O_ABORT = O_TMEM + 8, O_ABSENT = O_ABORT + 8,
                            O_PART = (O_ABSENT + RT_ABSENT * 4 + 15) & ~15u, O_STRIDES = O_PART + RT_PARTS * sizeof(RtPart),
                            O_DTAB = O_STRIDES + 32 * 4;
  static constexpr int DT_K = 16, DT_V = DT_K + 8 * KST, DT_N = DT_V + 8 * VST;   // descriptors: 8 per tile, Q_A, Q_B, K.., V..
  static_assert(O_DTAB + DT_N * 8 <= RT_CTRL, "control region too small");
  static_assert(DT_N <= RT_THREADS, "a thread per descriptor");
  static constexpr uint32_t O_Q = RT_CTRL, O_K = O_Q + 2 * TILE, O_V = O_K + KST * TILE, BYTES = O_V + VST * TILE;
  static_assert(BYTES <= 227 * 1024, "shared memory");
};

// fp32 accumulation, M = 128; B is MN-major for the product with V
constexpr uint32_t rt_idesc(bool fp16, int n, bool mn) {
  return (1u << 4) | (fp16 ? 0u : (1u << 7) | (1u << 10)) | (mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

struct RtSteps { uint64_t d[8]; };
// S = Q K^T: all descriptors are registers before the first MMA, so that the group leaves back to back
template <int KSTEPS>
__device__ __forceinline__ void rt_mma_qk(uint32_t s_tmem, const RtSteps& a, const RtSteps& b, uint32_t idesc) {
  if (KSTEPS == 8) {
    asm volatile(
        "{\n\t.reg .pred pz, po;\n\tsetp.ne.b32 pz, 0, 0;\n\tsetp.eq.b32 po, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %2, %10, %1, pz;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %3, %11, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %4, %12, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %13, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %6, %14, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %7, %15, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %8, %16, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %9, %17, %1, po;\n\t}"
        ::"r"(s_tmem), "r"(idesc),
          "l"(a.d[0]), "l"(a.d[1]), "l"(a.d[2]), "l"(a.d[3]), "l"(a.d[4]), "l"(a.d[5]), "l"(a.d[6]), "l"(a.d[7]),
          "l"(b.d[0]), "l"(b.d[1]), "l"(b.d[2]), "l"(b.d[3]), "l"(b.d[4]), "l"(b.d[5]), "l"(b.d[6]), "l"(b.d[7])
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred pz, po;\n\tsetp.ne.b32 pz, 0, 0;\n\tsetp.eq.b32 po, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %2, %6, %1, pz;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %3, %7, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %4, %8, %1, po;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %9, %1, po;\n\t}"
        ::"r"(s_tmem), "r"(idesc), "l"(a.d[0]), "l"(a.d[1]), "l"(a.d[2]), "l"(a.d[3]),
          "l"(b.d[0]), "l"(b.d[1]), "l"(b.d[2]), "l"(b.d[3])
        : "memory");
  }
}
// O (+)= P V, P at p_tmem + 8 i (16 packed columns per step)
__device__ __forceinline__ void rt_mma_pv(uint32_t o_tmem, uint32_t p_tmem, const RtSteps& v, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred pa, po;\n\tsetp.ne.b32 pa, %2, 0;\n\tsetp.eq.b32 po, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%3], %11, %1, pa;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%4], %12, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%5], %13, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%6], %14, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%7], %15, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%8], %16, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%9], %17, %1, po;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%10], %18, %1, po;\n\t}"
      ::"r"(o_tmem), "r"(idesc), "r"(acc),
        "r"(p_tmem), "r"(p_tmem + 8u), "r"(p_tmem + 16u), "r"(p_tmem + 24u), "r"(p_tmem + 32u), "r"(p_tmem + 40u),
        "r"(p_tmem + 48u), "r"(p_tmem + 56u),
        "l"(v.d[0]), "l"(v.d[1]), "l"(v.d[2]), "l"(v.d[3]), "l"(v.d[4]), "l"(v.d[5]), "l"(v.d[6]), "l"(v.d[7])
      : "memory");
}

// 32 bytes to a 32-byte boundary.  A thread writes its own row, so an instruction touches 32 lines whatever its width:
// half as many instructions are half the time (of 16-byte stores: 5% of a windowed prompt).
__device__ __forceinline__ void store_32(void* dst, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// P = 2^(s * scale - m) for 32 scores, packed in pairs; the unrounded weights are added to `sum`.  POLY of every 8 pairs
// are taken off the exponential unit (16 exponentials per clock and SM): a range reduction and a cubic on the FMA pipe.
//   u = sat((y + 127) / 255)        y = s * scale - m
//   n = round(255 u - 127) by the 1.5 * 2^23 trick;  f = 255 u - 127 - n in [-1/2, 1/2]
//   2^y = poly(f) * 2^n             n is added to the exponent field of poly(f)
// The cubic is the one of least relative error (1.02e-4, below the half step of either type by more than a factor of four) among
// those with poly(0) = 1.  That makes both ends of u exact: u = 0 leaves the bits of 1.0 less 127 exponents, which are those of
// 0, and u = 1 those of infinity.  So a masked score (-infinity) has the weight 0, whatever the value of its key - with 2^-57,
// where a range of [-57, 71] ended, a value of 1e20 that a token must not see was 690 in its output - and a score far above
// m shows in the sum.  Weights between 2^-127 and 2^-126 are rounded at will.
// Saturation makes 0 of NaN too, so `nan` says whether one of the polynomial's scores is NaN (it costs 1 - 2% at D = 64).
template <int POLY, bool FP16>
__device__ __forceinline__ void rt_weights(const uint32_t (&r)[32], float scale, float m, uint32_t (&pk)[16], float& sum, bool& nan) {
  float top = -INFINITY;
  const unsigned long long sc2 = f2_pack(scale, scale), nm2 = f2_pack(-m, -m);
  const float sc255 = scale * (1.f / 255.f), b255 = (127.f - m) * (1.f / 255.f);
  constexpr float MAGIC = 12582912.f - 127.f;      // 1.5 * 2^23 - 127
  const unsigned long long k255 = f2_pack(255.f, 255.f), kmag = f2_pack(MAGIC, MAGIC), kneg = f2_pack(-1.f, -1.f);
  const unsigned long long c0 = f2_pack(1.f, 1.f), c1 = f2_pack(0.6932829f, 0.6932829f), c2 = f2_pack(0.24221097f, 0.24221097f),
                           c3 = f2_pack(0.05500906f, 0.05500906f);
  unsigned long long acc[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float p0, p1;
    if (((j >> 1) & 7) < POLY) {
      top = max3_nan(top, __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
      const float u0 = __saturatef(fmaf(__uint_as_float(r[j]), sc255, b255));
      const float u1 = __saturatef(fmaf(__uint_as_float(r[j + 1]), sc255, b255));
      const unsigned long long u = f2_pack(u0, u1);
      const unsigned long long xf = f2_fma(u, k255, kmag);          // MAGIC + 127 + n (n in the low mantissa bits)
      const unsigned long long c = f2_fma(xf, kneg, kmag);          // -(127 + n)
      const unsigned long long f = f2_fma(u, k255, c);
      unsigned long long pl = f2_fma(f, c3, c2);
      pl = f2_fma(pl, f, c1);
      pl = f2_fma(pl, f, c0);
      float q0, q1, x0, x1;
      f2_unpack(pl, q0, q1);
      f2_unpack(xf, x0, x1);
      p0 = __uint_as_float(__float_as_uint(q0) + (__float_as_uint(x0) << 23));
      p1 = __uint_as_float(__float_as_uint(q1) + (__float_as_uint(x1) << 23));
    } else {
      const unsigned long long x = f2_pack(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
      float y0, y1;
      f2_unpack(f2_fma(x, sc2, nm2), y0, y1);
      p0 = fast_exp2(y0); p1 = fast_exp2(y1);
    }
    acc[(j >> 1) & 3] = f2_add(acc[(j >> 1) & 3], f2_pack(p0, p1));
    pk[j >> 1] = pack_half2<FP16>(p0, p1);
  }
  float a0, a1;
  f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), a0, a1);
  sum += a0 + a1;
  if (POLY > 0) nan |= top != top;
}

// the n lowest bits (n below 0: none, above 32: all)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

// The parts of items that a CTA runs through, in order, and the order of each part's units.
// A CTA that runs through the START of its last item takes the item's LAST units, and the next CTAs, which begin
// with the rest of it, take the units from the front; a whole item without a window starts at the unit whose
// number is that of units done (modulo those of the whole sequence), and wraps.  So CTAs that have done equally many
// units stand at about the same key of their items, and what one of them fetched the others find in L2.  (In the order of the keys, the last
// 2K chunk of a 34K prompt of 32 heads read its 143 MB of K and V 15 times from HBM: 2.1 GB.)
struct RtWalker {
  int req, head, tile, first, left, units, done;
  const int32_t* own;
  RaggedReq q;
  RaggedItem item;
  RaggedSpan span;
  __device__ void enter(const RaggedParams& p) {
    item = ragged_item(p, q, head, tile);
    span = ragged_span(p, q, tile);
    units = min(left, span.total - first);
  }
  __device__ bool begin(const RaggedParams& p, const RaggedStart& s, const int32_t* own_strides) {
    own = own_strides;
    req = s.req; head = s.head; tile = s.tile; first = s.first; left = s.units; done = 0; taken = s.taken;
    if (left <= 0) return false;
    q = ragged_req(p, req, own);
    enter(p);
    return true;
  }
  __device__ bool next(const RaggedParams& p) {
    left -= units; done += units;
    first = 0;
    if (left <= 0 || !ragged_next(p, req, head, tile, q, own)) return false;
    enter(p);
    return true;
  }
  __device__ void order(const RaggedParams& p, RtPart& part) const {
    const bool whole = units == span.total;
    // an item whose start an earlier CTA runs through: that one took the last units, this part's are that many earlier
    int from = first == 0 ? span.total - units : first - taken;
    if (whole) {
      from = p.window > 0 ? 0 : done % max((q.seq + RT_UNIT - 1) / RT_UNIT, 1);
      if (from >= span.total) from = 0;
    }
    part.units = units; part.whole = whole; part.slot = first == 0 ? 1 : 0;
    part.sink_units = min(max(span.sink_units - from, 0), units);
    part.embed = from == 0 ? span.embed : 0;
    part.sink_keys = span.sink_keys;
    if (from < span.sink_units) {             // sinks, then the window
      part.units_a = part.sink_units;
      part.key_a = from * RT_UNIT;
    } else {                                  // up to the end, then (a whole item) from the front
      part.units_a = min(span.total - from, units);
      part.key_a = span.win_key + (from - span.sink_units) * RT_UNIT;
    }
    part.key_b = span.win_key;
  }
  int taken;    // units of the CTA's first item that the CTA where it starts runs through
};

template <int D, bool FP16>
__global__ void __launch_bounds__(RT_THREADS, 1)
ragged_tc5_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k32,
                  const __grid_constant__ CUtensorMap map_v32, const __grid_constant__ RaggedParams p) {
  using C = RtCfg<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sbase = smem_addr(smem);
  const bool skewed = (sbase & 1023u) != 0;     // the swizzled tiles need a 1024-byte aligned base
  if (skewed || *reinterpret_cast<volatile unsigned int*>(&g_tc5_timeouts) > 16u) {
    if (threadIdx.x == 0) {
      if (skewed) atomicAdd(&g_tc5_timeouts, 1000u);
      ragged_wait_before();
      reinterpret_cast<RaggedStart*>(p.scratch)[blockIdx.x] = RaggedStart{};      // nothing for the join to read
    }
    return;
  }
  auto bar = [&](int b) { return sbase + 8u * uint32_t(b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::O_TMEM);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::O_ABORT);
  volatile uint32_t* absent_of = reinterpret_cast<volatile uint32_t*>(smem + C::O_ABSENT);
  uint64_t* dtab = reinterpret_cast<uint64_t*>(smem + C::O_DTAB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 64) { tma_prefetch_map(&map_q); tma_prefetch_map(&map_k); tma_prefetch_map(&map_v); }
  if (tid == 96) {
    for (int s = 0; s < RT_PARTS; ++s) { mbar_init(bar(C::B_PFULL + s), 1); mbar_init(bar(C::B_PEMPTY + s), 11); }
    for (int s = 0; s < C::KST; ++s) { mbar_init(bar(C::B_KFULL + s), 1); mbar_init(bar(C::B_KEMPTY + s), 2); }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(bar(C::B_VFULL + s), 1); mbar_init(bar(C::B_VEDGE + s), 1); mbar_init(bar(C::B_VEMPTY + s), 2);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(bar(C::B_QFULL + h), 1); mbar_init(bar(C::B_QEMPTY + h), 1);
      mbar_init(bar(C::B_SFULL + h), 1); mbar_init(bar(C::B_PREADY + h), 128); mbar_init(bar(C::B_ODONE + h), 1);
      mbar_init(bar(C::B_TOKEN + h), 1);
    }
    mbar_arrive(bar(C::B_TOKEN));     // stream A's thread goes first
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (tid >= RT_THREADS - C::DT_N) {
    const int e = tid - (RT_THREADS - C::DT_N), ks = e & 7;
    const uint64_t kstep = uint64_t(uint32_t(ks >> 2) * (RT_SLAB >> 4) + uint32_t(ks & 3) * (32u >> 4));
    if (e < C::DT_K) dtab[e] = desc_kmajor(sbase + C::O_Q + uint32_t(e >> 3) * C::TILE) + kstep;
    else if (e < C::DT_V) dtab[e] = desc_kmajor(sbase + C::O_K + uint32_t((e - C::DT_K) >> 3) * C::TILE) + kstep;
    else dtab[e] = desc_mnmajor(sbase + C::O_V + uint32_t((e - C::DT_V) >> 3) * C::TILE) + uint64_t(uint32_t(ks) * (2048u >> 4));
  }
  // Rows of the Q tiles that no copy fills (a group that does not divide 128) would be garbage, NaN perhaps, and a row whose
  // sum is not finite asks for a new reference point in every unit
  for (int e = p.stream_tokens * p.chunk_heads * 8 + tid; e < RT_ROWS * 8; e += RT_THREADS) {
#pragma unroll
    for (int s = 0; s < 2 * C::SLABS; ++s)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + C::O_Q + uint32_t(s) * RT_SLAB + uint32_t(e) * 16u), "r"(0) : "memory");
    fence_proxy_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // The producer finds the CTA's first part while the others set up: from here to the first scores is a chain of loads
  int32_t* sh_strides = reinterpret_cast<int32_t*>(smem + C::O_STRIDES);
  RtWalker w = {};
  RtPart part = {};
  bool more = false;
  int id = 0;
  const int box = p.copy_rows, per_unit = RT_UNIT / box;      // rows of a copy, copies of a unit and 64 columns
  const int my_col = lane % per_unit * box;
  // first key of this lane's copy of unit u, and its page (n_pages - behind the pool, zeros - where there is none)
  auto key_of = [&](int u) { return u == 0 && my_col < part.embed ? my_col : part.key0(u) + my_col; };
  auto page_of = [&](int u) {
    if (!p.table || u >= part.units) return 0;
    const int key = key_of(u);
    if (key >= w.span.keys) return p.n_pages;
    const int got = p.table[w.req * p.table_stride + (key >> p.page_shift)];
    return got >= 0 && got < p.n_pages ? got : p.n_pages;
  };
  if (warp == 0) {
    ragged_wait_before();
    const RaggedStart start = p.few ? ragged_start_few(p, blockIdx.x, lane, sh_strides)
                                    : reinterpret_cast<const RaggedStart*>(p.scratch)[blockIdx.x];
    __syncwarp();
    more = w.begin(p, start, sh_strides);
    if (more) {
      w.order(p, part);
      id = page_of(0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  RtPart* parts = reinterpret_cast<RtPart*>(smem + C::O_PART);
  // part n has been announced
  auto part_ready = [&](int n) { return mbar_wait(bar(C::B_PFULL + n % RT_PARTS), (n / RT_PARTS) & 1, abort_flag); };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(RT_REGS_CONTROL));
    if (warp == 0) {
      // ---------------------------------------------------------- producer (whole warp; lane 0 waits and announces)
      const int my_slab = lane / per_unit;
      const bool copies = my_slab < C::SLABS;
      const uint32_t my_dst = uint32_t(my_slab) * RT_SLAB + uint32_t(my_col) * 128u;
      const int in_page = p.table ? (1 << p.page_shift) - 1 : -1;
      const uint32_t q_bytes = uint32_t(p.stream_tokens * p.chunk_heads) * 128u * C::SLABS;
      auto wait0 = [&](int b, int parity) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait(bar(b), parity, abort_flag);
        return __shfl_sync(0xffffffffu, ok, 0);
      };
      auto load = [&](const CUtensorMap* map, int full, uint32_t tile, int key, int id, int kvh) {
        if (lane == 0) mbar_expect_tx(bar(full), C::TILE);
        __syncwarp();
        if (copies) tma_load_4d(tile + my_dst, map, bar(full), my_slab * 64, key & in_page, kvh, id);
      };
      // a unit of contiguous keys whose first columns are the keys from 0 on, 32 at a time
      auto load_embedded = [&](const CUtensorMap* map, int full, uint32_t tile, int key, int embed, int kvh) {
        if (lane == 0) mbar_expect_tx(bar(full), C::TILE);
        __syncwarp();
        const int col = (lane & 3) * 32, slab = lane >> 2;
        if (slab < C::SLABS)
          tma_load_4d(tile + uint32_t(slab) * RT_SLAB + uint32_t(col) * 128u, map, bar(full), slab * 64, col < embed ? col : key + col, kvh, 0);
      };
      int v_embed = 0;
      bool v_edge = false;
      uint32_t edges = 0, edge_last = 0;      // bits per V stage: parity of its edge units, whether its last unit was one
      int k_i = 0, v_i = 0, v_key = 0, v_id = 0, v_kvh = 0, pieces = 0;
      bool ok = true;
      auto load_v = [&]() {      // K runs one unit ahead of V
        const int s = v_i % C::VST;
        if (!wait0(C::B_VEMPTY + s, ((v_i / C::VST) & 1) ^ 1)) return false;
        const uint32_t tile = sbase + C::O_V + uint32_t(s) * C::TILE;
        const int full = (v_edge ? C::B_VEDGE : C::B_VFULL) + s;
        if (v_embed) load_embedded(&map_v32, full, tile, v_key, v_embed, v_kvh);
        else load(&map_v, full, tile, v_key, v_id, v_kvh);
        edges ^= uint32_t(v_edge) << s;
        edge_last = (edge_last & ~(1u << s)) | uint32_t(v_edge) << s;
        ++v_i;
        return true;
      };
      auto announce = [&](int n, const RtPart& part) {
        const bool free = wait0(C::B_PEMPTY + n % RT_PARTS, ((n / RT_PARTS) & 1) ^ 1);
        if (free && lane == 0) {
          parts[n % RT_PARTS] = part;
          mbar_arrive(bar(C::B_PFULL + n % RT_PARTS));
        }
        return free;
      };
      // a stream's Q tile is free when its last Q K^T of the previous part is done
      int q_n[2] = {0, 0};
      auto load_q = [&](int h) {
        if (q_n[h] > 0 && !wait0(C::B_QEMPTY + h, (q_n[h] - 1) & 1)) return false;
        if (lane == 0) {
          mbar_expect_tx(bar(C::B_QFULL + h), q_bytes);
          for (int s = 0; s < C::SLABS; ++s)
            tma_load_3d(sbase + C::O_Q + uint32_t(h) * C::TILE + uint32_t(s) * RT_SLAB, &map_q, bar(C::B_QFULL + h), s * 64,
                        w.item.kvh * p.group + w.item.h0, w.q.row0 + w.item.tok0 + h * p.stream_tokens);
        }
        ++q_n[h];
        return true;
      };
      while (ok && more) {
        part.both = w.item.n_tok > p.stream_tokens;
        part.n_tok = w.item.n_tok; part.heads = w.item.heads; part.pos0 = w.item.pos0; part.keys = w.span.keys;
        part.low = p.window > 0 ? w.item.pos0 - p.window + 1 : 0;
        part.out = ragged_out(p, w.q, w.item, 0, 0, D);
        ok = announce(pieces, part);
        // Q before the first K unit: the other way round a windowed prompt takes 4% longer
        if (ok) ok = load_q(0) && (!part.both || load_q(1));
        if (!ok) break;
        for (int u = 0; u < part.units; ++u) {
          const int key = key_of(u), id_next = page_of(u + 1);
          const int s = k_i % C::KST;
          ok = wait0(C::B_KEMPTY + s, ((k_i / C::KST) & 1) ^ 1);
          if (!ok) break;
          // pages that the sequence should have here and has not: a bit per 16 keys
          const unsigned gone = p.table ? __ballot_sync(0xffffffffu, lane < per_unit && id == p.n_pages) : 0u;
          if (lane == 0) {
            uint32_t bits = 0;
            for (int g = 0; gone && g < per_unit; ++g)
              if (gone >> g & 1u) bits |= ((1u << (box >> 4)) - 1u) << (g * (box >> 4));
            absent_of[k_i % RT_ABSENT] = bits;
            __threadfence_block();
          }
          const int embed = !p.table && u == 0 ? part.embed : 0;
          if (embed) load_embedded(&map_k32, C::B_KFULL + s, sbase + C::O_K + uint32_t(s) * C::TILE, part.key_a, embed, w.item.kvh);
          else load(&map_k, C::B_KFULL + s, sbase + C::O_K + uint32_t(s) * C::TILE, key, id, w.item.kvh);
          ++k_i;
          if (u > 0) ok = load_v();
          if (!ok) break;
          v_embed = embed;
          v_edge = part.edge(u);
          v_key = embed ? part.key_a : key; v_id = id; v_kvh = w.item.kvh;
          id = id_next;
        }
        if (ok) ok = load_v();
        ++pieces;
        more = w.next(p);
        if (more) {
          w.order(p, part);
          id = page_of(0);
        }
      }
      if (ok) {
        part.units = 0;
        announce(pieces, part);
      }
      // every copy that was started must have landed before the CTA may exit
      if (lane == 0) {
        for (int h = 0; h < 2; ++h)
          if (q_n[h] > 0) mbar_wait(bar(C::B_QFULL + h), (q_n[h] - 1) & 1, abort_flag, true);
        for (int j = max(0, k_i - C::KST); j < k_i; ++j) mbar_wait(bar(C::B_KFULL + j % C::KST), (j / C::KST) & 1, abort_flag, true);
        for (int j = max(0, v_i - C::VST); j < v_i; ++j) {
          const int s = j % C::VST;
          if (edge_last >> s & 1u) mbar_wait(bar(C::B_VEDGE + s), (edges >> s & 1u) ^ 1u, abort_flag, true);
          else mbar_wait(bar(C::B_VFULL + s), (j / C::VST) & 1, abort_flag, true);
        }
      }
    } else if (warp <= 2) {
      // ---------------------------------------------------------- MMA issuers
      if (lane == 0) {
        const int h = warp - 1;
        const uint32_t ts = tmem + (h == 0 ? 0u : 128u), to = tmem + 256u + uint32_t(h) * D, tp = C::P_BESIDE ? tmem + 384u + uint32_t(h) * 64u : ts;
        constexpr uint32_t ID_QK = rt_idesc(FP16, 128, false), ID_PV = rt_idesc(FP16, D, true);
        auto fetch = [&](int first, RtSteps& o) {
          const ulonglong2* src = reinterpret_cast<const ulonglong2*>(dtab + first);
#pragma unroll
          for (int j = 0; j < 4; ++j) { const ulonglong2 t = src[j]; o.d[2 * j] = t.x; o.d[2 * j + 1] = t.y; }
        };
        auto release = [&](int b, bool used) { if (used) tc_commit(bar(b)); else mbar_arrive(bar(b)); };
        int step = 0, i = 0, np = 0, nq = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
          ok = part_ready(n);
          if (!ok) break;
          const int units = parts[n % RT_PARTS].units;
          const bool both = parts[n % RT_PARTS].both != 0, mine = h == 0 || both;
          mbar_arrive(bar(C::B_PEMPTY + n % RT_PARTS));
          if (units == 0) break;
          // Step u: P V of unit u and Q K^T of unit u + 1, the two groups back to back.  Step -1 has only the latter and
          // takes no turn: stream A's next item must not wait for stream B's last softmax
          if (mine) ok = mbar_wait(bar(C::B_QFULL + h), nq++ & 1, abort_flag);
          for (int u = -1; ok && u < units; ++u) {
            const bool pv = u >= 0, qk = u + 1 < units;
            const int vs = (i + C::VST - 1) % C::VST, ks = i % C::KST;     // i: units of the CTA whose Q K^T has been issued
            if (pv) ok = mbar_wait(bar(C::B_VFULL + vs), ((i - 1) / C::VST) & 1, abort_flag);
            if (ok && qk) ok = mbar_wait(bar(C::B_KFULL + ks), (i / C::KST) & 1, abort_flag);
            if (!ok) break;
            if (mine) {
              RtSteps vd, qd, kd;
              if (pv) fetch(C::DT_V + 8 * vs, vd);
              if (qk) { fetch(8 * h, qd); fetch(C::DT_K + 8 * ks, kd); }
              if (both && pv) ok = mbar_wait(bar(C::B_TOKEN + h), step & 1, abort_flag);
              if (ok && pv) ok = mbar_wait(bar(C::B_PREADY + h), np & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              if (pv) {
                rt_mma_pv(to, tp, vd, ID_PV, u > 0 ? 1u : 0u);
                ++np;
                if (!qk) tc_commit(bar(C::B_ODONE + h));
              }
              if (qk) { rt_mma_qk<C::KSTEPS>(ts, qd, kd, ID_QK); tc_commit(bar(C::B_SFULL + h)); }
              if (both && pv) { mbar_arrive(bar(C::B_TOKEN + (h ^ 1))); ++step; }
            }
            if (pv) release(C::B_VEMPTY + vs, mine);
            if (qk) {
              release(C::B_KEMPTY + ks, mine);
              if (mine && u + 2 == units) tc_commit(bar(C::B_QEMPTY + h));
              ++i;
            }
          }
        }
      }
    } else {
      // ---------------------------------------------------------- V rows that no query of the item sees become zeros
      // (such a unit's copies complete on a barrier of their own, and this warp's arrival makes the unit full)
      bool ok = true;
      int i = 0;
      uint32_t edges = 0;       // a bit per stage: parity of its edge units
      for (int n = 0; ok; ++n) {
        ok = __all_sync(0xffffffffu, part_ready(n));
        if (!ok) break;
        const RtPart part = parts[n % RT_PARTS];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::B_PEMPTY + n % RT_PARTS));
        if (part.units == 0) break;
        for (int u = 0; u < part.units; ++u, ++i) {
          if (!part.edge(u)) continue;
          const int s = i % C::VST;
          ok = __all_sync(0xffffffffu, mbar_wait(bar(C::B_VEDGE + s), edges >> s & 1u, abort_flag));
          if (!ok) break;
          edges ^= 1u << s;
          const int key = part.key0(u);
          const int tail = min(max(part.keys - key, 0), RT_UNIT);                                       // rows [tail, 128)
          const int embed = u == 0 ? part.embed : 0;                                                    // rows [sink_keys, embed)
          const int a = max(min(max(p.sinks - key, 0), RT_UNIT), embed), b = min(max(part.low - key, 0), tail);   // and [a, b)
          const uint32_t base = sbase + C::O_V + uint32_t(s) * C::TILE;
          for (int r = lane >> 3; r < RT_UNIT; r += 4)
            if (r >= tail || (r >= a && r < b) || (r >= part.sink_keys && r < embed))
#pragma unroll
              for (int sl = 0; sl < C::SLABS; ++sl)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                             ::"r"(base + uint32_t(sl) * RT_SLAB + uint32_t(r) * 128u + uint32_t(lane & 7) * 16u), "r"(0) : "memory");
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(C::B_VFULL + s));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax warpgroups
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(RT_REGS_SOFTMAX));
    // Weights are 2^LIFT times what the reference point says, and a unit's sum of them above SUM_LIMIT moves the point to the
    // unit's maximum.  The factor cancels in O / l, and all parts of an item have it.
    //   bf16: O, the sum of weight times value, must not overflow with values up to 3.4e38, so weights are 2^-32 and less at
    //         first, and a unit's sum stays below 2^-8 (without this a score that rose by 2^60 overflowed with values of 1e25)
    //   fp16: P reaches 65504 only, and the multiples of 2^-24 that small weights are rounded to should be small against the
    //         largest weight: at 2^8 (128 of them are below the limit) they lose 2^-33 of it per key, not 2^-25, which over
    //         100K keys behind one that all tokens look at was 0.4% of the mass
    constexpr float SUM_LIMIT = FP16 ? 61440.f : 0.00390625f, MARGIN = FP16 ? 0.f : 12.f, LIFT = FP16 ? 8.f : -32.f;
    // The 128 scores of a row and the constants of the exponentials leave about twenty registers: what the loop over
    // units does not need is looked up (in shared memory) or computed again where it is used.
    const int h = (warp - 4) >> 2;
    const uint32_t tS = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(h * 128);
    auto p_tmem = [&]() { return tS + (C::P_BESIDE ? 384u - uint32_t(h) * 64u : 0u); };     // 384 + 64 h, or S itself
    auto o_tmem = [&]() { return tmem + (uint32_t((warp & 3) * 32) << 16) + 256u + uint32_t(h) * D; };
    // this thread's row: token of the item, head of the chunk, and whether the item has it
    struct Place { int tok, head; bool in; };
    auto place = [&](const volatile RtPart& part) {
      const int row = (warp & 3) * 32 + lane, t = row / p.chunk_heads;
      Place x;
      x.head = row - t * p.chunk_heads;
      x.tok = h * p.stream_tokens + t;
      x.in = t < p.stream_tokens && x.tok < part.n_tok && x.head < part.heads;
      return x;
    };
    // bit 0: units of this stream, bit 1: its items, bits 2, 3: parts, from bit 4: units of the CTA (the first three
    // wrap, which is all that the barriers' phases need)
    uint32_t seen_so_far = 0;
    bool ok = true;
    while (true) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar(C::B_PFULL + int(seen_so_far >> 2 & 1u)), seen_so_far >> 3 & 1u, abort_flag));
      if (!ok) break;
      const volatile RtPart& part = parts[seen_so_far >> 2 & 1u];
      auto part_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::B_PEMPTY + int(seen_so_far >> 2 & 1u)));
        seen_so_far = (seen_so_far & ~12u) | ((seen_so_far + 4u) & 12u);
      };
      if (part.units == 0) { part_done(); break; }
      if (h == 1 && !part.both) { seen_so_far += uint32_t(part.units) << 4; part_done(); continue; }
      float m_used = -INFINITY, l_sum = 0.f;
      bool fresh = true;                     // some row of the warp has seen no key yet
      for (int u = 0; u < part.units; ++u) {
        const int key = u < part.units_a ? part.key_a + u * RT_UNIT : part.key_b + (u - part.units_a) * RT_UNIT;
        // seen whole by every row of the stream: up to its first token's position, from its last token's window on
        const int first_pos = part.pos0 + h * p.stream_tokens;
        const bool past = key + RT_UNIT - 1 > first_pos, before = p.window > 0 && key < first_pos + p.stream_tokens - p.window;
        ok = __all_sync(0xffffffffu, mbar_wait(bar(C::B_SFULL + h), seen_so_far & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        // Masking rewrites S in TMEM, 32 columns at a time, before the row is read: kept apart like this it costs the
        // units that need none nothing but the branch (masks on the row's registers cost them 6%).
        const uint32_t gone = absent_of[(seen_so_far >> 4) % RT_ABSENT];
        if (past || before || gone != 0u) {
          const Place x = place(part);
          const int row_last = (x.in ? part.pos0 + x.tok : -1) - key;    // last column the row sees
          const int last = u < part.sink_units ? min(row_last, part.sink_keys - 1 - key) : row_last;
          const int a = max(p.sinks - key, 0), b = before ? row_last - p.window + 1 : 0;    // and not [a, b)
          const int embed = u == 0 ? part.embed : 0, sinks = x.in ? part.sink_keys : 0;     // columns of the first keys, those that count
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const uint32_t bad = (gone >> (2 * c) & 1u ? 0xffffu : 0u) | (gone >> (2 * c + 1) & 1u ? 0xffff0000u : 0u);
            const uint32_t firsts = low_bits(embed - c * 32);
            const uint32_t keep = ((low_bits(last + 1 - c * 32) & ~(low_bits(b - c * 32) & ~low_bits(a - c * 32)) & ~firsts) |
                                   (low_bits(sinks - c * 32) & firsts)) & ~bad;
            if (__any_sync(0xffffffffu, keep != 0xffffffffu)) {
              float v[32];
              tmem_ld32(tS + c * 32, v);
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(keep >> j & 1u)) v[j] = -INFINITY;
              tmem_st32(tS + c * 32, v);
            }
          }
          tc_wait_st();
        }
        auto row_max_log2 = [&]() {
          float m = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t r[32];
            tmem_ld32_raw(tS + c * 32, r);
            tc_wait_ld();
            m = fmaxf(m, row_max(r));
          }
          return m * p.scale_log2;
        };
        // a row's reference is the maximum of the first unit in which it sees a key (nothing was added before)
        if (fresh) {
          const float mb = row_max_log2();
          if (m_used == -INFINITY) m_used = mb;
          if (mb == INFINITY) l_sum = NAN;       // infinity less itself
          fresh = __any_sync(0xffffffffu, m_used == -INFINITY);
        }
        // S must stay in TMEM until the row's sum has been looked at, for the case that the reference has to move.  At D = 64
        // there is room for P beside it; at D = 128 P is held in registers and then written over S.  Either way no more than
        // three quarters of S are in registers.
        uint32_t pk0[16], pk1[16], pk2[16], pk3[16];
        float blk;
        bool moved = u == 0;
        while (true) {
          const float ref = m_used == -INFINITY ? 0.f : m_used - LIFT;
          blk = 0.f;
          bool nan = false;
          uint32_t s0[32], s1[32], s2[32], s3[32];
          tmem_ld32_raw(tS + 0, s0);
          tmem_ld32_raw(tS + 32, s1);
          tc_wait_ld();
          tmem_ld32_raw(tS + 64, s2);
          rt_weights<C::POLY, FP16>(s0, p.scale_log2, ref, pk0, blk, nan);
          if (C::P_BESIDE) tmem_st16(p_tmem(), pk0);
          tmem_ld32_raw(tS + 96, s3);
          rt_weights<C::POLY, FP16>(s1, p.scale_log2, ref, pk1, blk, nan);
          if (C::P_BESIDE) tmem_st16(p_tmem() + 16, pk1);
          tc_wait_ld();
          rt_weights<C::POLY, FP16>(s2, p.scale_log2, ref, pk2, blk, nan);
          if (C::P_BESIDE) tmem_st16(p_tmem() + 32, pk2);
          rt_weights<C::POLY, FP16>(s3, p.scale_log2, ref, pk3, blk, nan);
          if (C::P_BESIDE) tmem_st16(p_tmem() + 48, pk3);
          if (nan) blk = NAN;
          if (moved || !__any_sync(0xffffffffu, !(blk <= SUM_LIMIT))) break;
          moved = true;
          const float mb = row_max_log2();
          float alpha = 1.f;
          if (mb > m_used + MARGIN) {
            alpha = exp2f(m_used - mb);
            m_used = mb;
            l_sum *= alpha;
            if (mb == INFINITY) l_sum = NAN;
          }
          // S of this unit is complete, hence so is every earlier P V of the stream: O is stable
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float v[32];
            tmem_ld32(o_tmem() + c * 32, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= alpha;
            tmem_st32(o_tmem() + c * 32, v);
          }
        }
        if (!C::P_BESIDE) {
          tmem_st16(p_tmem(), pk0); tmem_st16(p_tmem() + 16, pk1); tmem_st16(p_tmem() + 32, pk2); tmem_st16(p_tmem() + 48, pk3);
        }
        l_sum += blk;
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(bar(C::B_PREADY + h));
        seen_so_far = (seen_so_far ^ 1u) + 16u;
      }
      // ---- epilogue: the row goes to the output, or with its statistics to the scratch
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(C::B_ODONE + h), seen_so_far >> 1 & 1u, abort_flag));
      if (!ok) break;
      seen_so_far ^= 2u;
      tc_fence_after();
      const Place x = place(part);
      if (part.whole) {
        const float inv = l_sum == 0.f ? 0.f : 1.f / l_sum;     // (no key: 0; a NaN stays one)
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (x.in ? part.out + (int64_t(x.tok) * p.n_q_heads + x.head) * D : 0);
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t r0[32], r1[32];
          tmem_ld32_raw(o_tmem() + c * 64, r0);
          tmem_ld32_raw(o_tmem() + c * 64 + 32, r1);
          tc_wait_ld();
          if (x.in) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t* v = j < 2 ? r0 + 16 * j : r1 + 16 * (j - 2);
                o[e] = pack_half2<FP16>(__uint_as_float(v[2 * e]) * inv, __uint_as_float(v[2 * e + 1]) * inv);
              }
              store_32(dst + c * 64 + j * 16, o);
            }
          }
        }
      } else {
        float* dst_part = ragged_part(p, blockIdx.x, part.slot, D);
        const int at = h * RT_ROWS + (warp & 3) * 32 + lane;
        if (x.in) { dst_part[at] = m_used; dst_part[2 * RT_ROWS + at] = l_sum; }
        float* dst = dst_part + 4 * RT_ROWS + at * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          tmem_ld32(o_tmem() + c * 32, v);
          if (x.in) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(v[8 * j + e]);
              store_32(dst + c * 32 + j * 8, o);
            }
          }
        }
      }
      tc_fence_before();     // the next item's first P (after its S) lets the next product overwrite O
      part_done();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// ---------------------------------------------------------------- host side
void ragged_tc5_config(RaggedParams& p) {
  p.head_chunks = ceil_div(p.group, RT_ROWS);
  p.chunk_heads = ceil_div(p.group, p.head_chunks);
  p.stream_rows = RT_ROWS;
  p.stream_tokens = RT_ROWS / p.chunk_heads;
  p.tile_rows = 2 * RT_ROWS;
  p.tile_tokens = 2 * p.stream_tokens;
  p.unit_shift = 7;
  static_assert(RT_UNIT == 128, "keys of a unit");
  // A copy is a page or 128 keys; the unit of contiguous keys in which sinks stand first is copied 32 keys at a time
  const int page = 1 << p.page_shift;
  p.copy_rows = p.table && page < RT_UNIT ? page : RT_UNIT;
  p.granule = p.table ? p.copy_rows : p.window > 0 && p.sinks > 0 ? 32 : 16;
  p.n_ctas = RT_CTAS;
}

static bool tma_stride(int64_t s) { return s > 0 && s * 2 < (int64_t(1) << 40); }

// a stride of a dimension of extent one is never used and may be anything
bool ragged_tc5_describable(const RaggedParams& p) {
  const bool one_head = p.n_kv_heads == 1, one_page = p.n_pages == 1;
  return (p.n_rows == 1 || tma_stride(p.q_sn)) && (p.n_q_heads == 1 || tma_stride(p.q_sh)) && tma_stride(p.k_st) && tma_stride(p.v_st) &&
         (one_head || (tma_stride(p.k_sh) && tma_stride(p.v_sh))) && (!p.table || one_page || (tma_stride(p.k_sp) && tma_stride(p.v_sp)));
}

// K or V as (d, token of the page, head, page); contiguous keys are one page
static bool rt_map_kv(CUtensorMap* m, const RaggedParams& p, const void* base, int64_t sp, int64_t st, int64_t sh, int d, int rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int page = p.table ? 1 << p.page_shift : p.seq_one;
  const cuuint64_t dims[4] = {cuuint64_t(d), cuuint64_t(page), cuuint64_t(p.n_kv_heads), cuuint64_t(p.n_pages)};
  const cuuint64_t strides[3] = {cuuint64_t(st) * 2, cuuint64_t(p.n_kv_heads == 1 ? d : sh) * 2,
                                 cuuint64_t(!p.table || p.n_pages == 1 ? d : sp) * 2};
  const cuuint32_t box[4] = {64, cuuint32_t(rows), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, p.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Q as (d, head, token): a copy of chunk_heads x stream_tokens rows lands as one tile, token by token
static bool rt_map_q(CUtensorMap* m, const RaggedParams& p, int d) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(p.n_q_heads), cuuint64_t(p.n_rows)};
  const cuuint64_t strides[2] = {cuuint64_t(p.n_q_heads == 1 ? d : p.q_sh) * 2, cuuint64_t(p.n_rows == 1 ? d : p.q_sn) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(p.chunk_heads), cuuint32_t(p.stream_tokens)};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, p.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p.q), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool FP16>
static int launch_tc5(const RaggedParams& p, cudaStream_t st) {
  CUtensorMap mq, mk, mv, mk32, mv32;
  if (!rt_map_q(&mq, p, D) || !rt_map_kv(&mk, p, p.k, p.k_sp, p.k_st, p.k_sh, D, p.copy_rows) ||
      !rt_map_kv(&mv, p, p.v, p.v_sp, p.v_st, p.v_sh, D, p.copy_rows))
    return SPF_ERR_SHAPE;
  mk32 = mk; mv32 = mv;
  if (!p.table && p.granule == 32 &&
      (!rt_map_kv(&mk32, p, p.k, p.k_sp, p.k_st, p.k_sh, D, 32) || !rt_map_kv(&mv32, p, p.v, p.v_sp, p.v_st, p.v_sh, D, 32)))
    return SPF_ERR_SHAPE;
  const cudaError_t e = cudaFuncSetAttribute(ragged_tc5_kernel<D, FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(RtCfg<D>::BYTES));
  if (e != cudaSuccess) { note_cuda_error(e); return SPF_ERR_LAUNCH; }
  return ragged_launch_after(ragged_tc5_kernel<D, FP16>, dim3(p.n_ctas), RT_THREADS, int(RtCfg<D>::BYTES), st, mq, mk, mv, mk32, mv32, p);
}

int ragged_tc5_attention(const RaggedParams& p, int head_dim, cudaStream_t st) {
  if (head_dim == 128) return p.fp16 ? launch_tc5<128, true>(p, st) : launch_tc5<128, false>(p, st);
  return p.fp16 ? launch_tc5<64, true>(p, st) : launch_tc5<64, false>(p, st);
}

unsigned int ragged_tc5_timeout_count() { return tc5_read_timeouts_here(); }
bool ragged_tc5_reset_timeouts() { return tc5_reset_timeouts_here(); }
bool ragged_tc5_set_wait_limit(unsigned long long ns) { return tc5_set_wait_limit_here(ns); }

}  // namespace spf
