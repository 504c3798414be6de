// Products of few rows with 4-bit expert weights (moe_rd_expert_matvec_w4):
//   out[r,n] = sum_groups scale[n,group] * sum_{k in group} x[r,k] * (q[n,k] - zero[n,group])
//
// Reading the weights (half a byte each) of the experts that have rows is nearly all the traffic, so HBM is the floor:
// 43 bytes, 87 weights, per nanosecond and SM.  A product on the CUDA cores would need one FMA per weight and row; from
// two rows on that is slower than the memory.  So the weights go through the warp's matrix instruction (mma m16n8k16: 16
// outputs x 16 inputs times 8 rows of x), and what has to be kept small is the number of instructions that turn 4-bit
// integers into its operands:
//
// * A tile of 32 outputs x 128 inputs is 2 KB, stored so that a lane's 16-byte loads are its operand fragments: word i
//   holds the eight inputs 32i + 8j.. of one output, the pair (2p, 2p+1) in nibble p of its two halves.
// * bf16: (w >> 4p) & 0x000f000f with the exponent of 128 or'ed in (one LOP3) is the pair 128 + q, from which 128 + zero is
//   subtracted exactly: q - zero is an integer in -15..15.
// * fp16: there is room for two nibbles below the exponent, 1024 + q and 1024 + 16 q, from which a subtraction or a fused
//   multiply-add makes q - zero exactly: a third of the shifts.
// * The scale of a group multiplies its fp32 sum; nothing is rounded below 32 bits before the result is.
// Leaving the subtraction to the sums (operands 128 + q or 16 + q, and (16 + zero) * sum of x taken off afterwards) saves a
// quarter of the instructions and was slower: the sums of x cost matrix instructions, and it is their chains that a warp
// waits for (8 experts x 8192 outputs x 7168 inputs 51.3 against 50.3 us; groups of 32 64.5 against 54.4 us).
// The copies alone run at 6.7 TB/s (64 experts x 4096 x 7168: 145 us), the kernel at 5.5 (175 us): what bounds it is the
// integer pipe, 7 instructions for 8 bf16 weights (5 for fp16, 6 % faster).
//
// A unit of work is 32 outputs of one expert for up to eight of its rows (or 16, see launch_w4_rows); its tiles lie one
// behind the other in memory, and so do the units of an expert.  Only experts that have rows get units: every block lists
// them from the offsets.  A block gets a run of whole units, and its warps equal shares of the run's tiles, cut anywhere: a
// warp streams one contiguous stretch of weights, kDepth tiles ahead of its products (cp.async into its own part of
// shared memory; it waits for nothing but its own copies), writes the units that it has from end to end, and leaves the
// sums of the cut ones (at most its first and its last) in shared memory, where after a barrier they are added in the
// warps' order.
#include <atomic>

#include "row_types.cuh"

namespace moe_rd {

int device_sms();

namespace {

constexpr int kW4Threads = 512;
constexpr int kW4Warps = kW4Threads / 32;
// Tiles in flight per warp while another is being multiplied: 2 KB x 16 warps is 32 KB an SM, most of a microsecond of its
// share of the HBM rate.  Deeper rings are slower: 64 experts x 4096 outputs x 7168 inputs, one row each, 175 us with 1, 181
// with 2; 8 experts x 2048 outputs 17.8, 18.4 us.
constexpr int kDepth = 1;
constexpr int kTileBytes = 2048;

struct W4Args {
  const unsigned char* x;
  const unsigned char* weight;
  const unsigned char* scales;
  const unsigned char* zeros;
  const int32_t* offsets;
  unsigned char* out;
  int64_t rows;
  int N, K, E, G;
  int chunks;   // tiles of 128 inputs
  int nblocks;  // blocks of 32 outputs
  uint32_t group_magic;  // ceil(2^32 / (group / 32)): b / (group / 32) = (b * group_magic) >> 32 for b < 2^16; 0: group = 32
};

// SPAN: blocks of 32 inputs of a tile that share a group's scale: 4 (groups of a multiple of 128), 2 (64) or 1.
template <int SPAN, bool ZEROS>
struct W4Stage {
  static constexpr int kParts = 4 / SPAN;                     // groups in a tile
  static constexpr int kScales = kTileBytes;                  // [parts][8] four scales (outputs g, g + 8, g + 16, g + 24)
  static constexpr int kZeros = kScales + 64 * kParts;        // [parts][8] their zero points, four bits each
  static constexpr int kBytes = kZeros + (ZEROS ? 16 * kParts : 0);
};

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
  return r;
}

// A constant that the compiler keeps in a register (LOP3 takes one immediate, not two).
template <uint32_t V>
__device__ __forceinline__ uint32_t in_register() {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "n"(V));
  return r;
}

template <int DT>
struct W4Type;

template <>
struct W4Type<MOE_RD_T_BF16> {
  uint32_t mask = in_register<0x000f000fu>(), base = in_register<0x43004300u>();
  static __device__ __forceinline__ float first(uint32_t v) { return bf16_lo(v); }
  static __device__ __forceinline__ float second(uint32_t v) { return bf16_hi(v); }
  static __device__ __forceinline__ uint32_t zero_operand(uint32_t zero) { return 0x43004300u | (zero * 0x00010001u); }
  // the four operands q - zero of a word
  __device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&o)[4]) const {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t v = and_or(w >> (4 * p), mask, base);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&zero));
      o[p] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
  static __device__ __forceinline__ uint16_t round(float v) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<const uint16_t*>(&b);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};

template <>
struct W4Type<MOE_RD_T_FP16> {
  uint32_t low = in_register<0x000f000fu>(), high = in_register<0x00f000f0u>(), base = in_register<0x64006400u>();
  static __device__ __forceinline__ float first(uint32_t v) { return __low2float(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ float second(uint32_t v) { return __high2float(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ uint32_t zero_operand(uint32_t zero) { return 0x64006400u | (zero * 0x00010001u); }
  __device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&o)[4]) const {
    const uint32_t v = w >> 8;
    // 1024 + zero -> -(64 + zero): the same bits of zero, sixteen times as high in the mantissa
    const uint32_t z16 = ((zero & 0x000f000fu) << 4) | 0xd400d400u;
    const uint32_t e[4] = {and_or(w, low, base), and_or(w, high, base), and_or(v, low, base), and_or(v, high, base)};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const __half2 h = *reinterpret_cast<const __half2*>(&e[p]);
      const __half2 d = p & 1 ? __hfma2(h, __float2half2_rn(0.0625f), *reinterpret_cast<const __half2*>(&z16))
                              : __hsub2(h, *reinterpret_cast<const __half2*>(&zero));
      o[p] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
  static __device__ __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};

// acc += the product of one tile: w[2s + h] are the words of outputs 16s + 8h + g, x(q, v) the lane's inputs of block q for
// rows 8v.., scale(k, i) and zero(k, i) those of group k of the tile and output 8i + g.
template <int DT, int SPAN, int NT, typename X, typename Scale, typename Zero>
__device__ __forceinline__ void w4_tile(const W4Type<DT>& ty, const uint4 (&w)[4], X x, Scale scale, Zero zero,
                                        float (&acc)[2][NT][4]) {
  using Ty = W4Type<DT>;
  const uint32_t word[4][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w},
                               {w[2].x, w[2].y, w[2].z, w[2].w}, {w[3].x, w[3].y, w[3].z, w[3].w}};
#pragma unroll
  for (int k = 0; k < 4 / SPAN; ++k) {
    float part[2][NT][4];
#pragma unroll
    for (int q = k * SPAN; q < (k + 1) * SPAN; ++q) {
      uint4 xq[NT];
#pragma unroll
      for (int v = 0; v < NT; ++v) xq[v] = x(q, v);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint32_t a[4], b[4];
        ty.unpack(word[2 * s][q], zero(k, 2 * s), a);
        ty.unpack(word[2 * s + 1][q], zero(k, 2 * s + 1), b);
#pragma unroll
        for (int v = 0; v < NT; ++v) {
          float(&d)[4] = part[s][v];
          if (q == k * SPAN)
            Ty::mma(d, a[0], b[0], a[1], b[1], xq[v].x, xq[v].y, 0.0f, 0.0f, 0.0f, 0.0f);
          else
            Ty::mma(d, a[0], b[0], a[1], b[1], xq[v].x, xq[v].y, d[0], d[1], d[2], d[3]);
          Ty::mma(d, a[2], b[2], a[3], b[3], xq[v].z, xq[v].w, d[0], d[1], d[2], d[3]);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int v = 0; v < NT; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[s][v][i] = fmaf(scale(k, 2 * s + (i >> 1)), part[s][v][i], acc[s][v][i]);
  }
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// 8 bytes, of which the first `bytes` (0 or 8) are read and the rest become zero
__device__ __forceinline__ void copy8(uint32_t to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

__device__ __forceinline__ uint32_t w4_group(const W4Args& a, uint32_t b) {  // of block b of 32 inputs; G or more: padding
  return a.group_magic != 0 ? __umulhi(b, a.group_magic) : b;
}

// The lane's inputs of block q of tile c, from where its inputs of the tile begin; zeros past the last input.
__device__ __forceinline__ uint4 w4_load_x(const W4Args& a, const unsigned char* xp, int c, int q) {
  return 128 * c + 32 * q < a.K ? __ldg(reinterpret_cast<const uint4*>(xp + 64 * q)) : make_uint4(0u, 0u, 0u, 0u);
}

// ... of all its blocks; only the last tile can have padding.
__device__ __forceinline__ void w4_load_x(const W4Args& a, const unsigned char* xp, int c, uint4 (&x)[4]) {
  if (c < a.K >> 7) {
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = __ldg(reinterpret_cast<const uint4*>(xp + 64 * q));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = w4_load_x(a, xp, c, q);
  }
}

// Where a warp is in its share of the block's tiles.
struct W4Place {
  int i, nb, pass;  // expert (of the list), block of 32 outputs, pass over 8 * NT rows
  int c;            // tile of 128 inputs
};

// What a warp has left in shared memory: the part of a unit that an earlier warp began, with or without its end, and the
// part of a unit that it began itself and later warps end.
enum { kContinues = 1, kEnds = 2, kBegins = 4 };

template <int NT>
struct W4Joint {
  float sum[2 * kW4Warps][256 * NT];  // [warp]: the part of the first unit; [kW4Warps + warp]: of the last; [row of x][output]
  W4Place place[kW4Warps];          // of the unit that the warp began
  int what[kW4Warps];
  int expert[kMaxE], lo[kMaxE], n[kMaxE], unit[kMaxE];  // experts that have rows: number, rows, units before
};

// The units that several warps have: a thread per sum, 256 NT a unit, added in the order of the warps.
template <int DT, int NT>
__device__ __forceinline__ void w4_join(const W4Args& a, const W4Joint<NT>& s) {
  constexpr int kSums = 256 * NT;
  const int tid = threadIdx.x, lane = tid & 31;
  const int what = lane < kW4Warps ? s.what[lane] : 0;
  const unsigned continues = __ballot_sync(kFull, what & kContinues), ends = __ballot_sync(kFull, what & kEnds);
  unsigned begins = __ballot_sync(kFull, what & kBegins);
  for (int k = 0; begins != 0; ++k, begins &= begins - 1) {
    if (k % (kW4Threads / kSums) != tid / kSums) continue;
    const int w = __ffs(begins) - 1;
    const int last = w + __ffs(ends >> (w + 1));
    const W4Place p = s.place[w];
    const int el = tid & (kSums - 1), r = p.pass * 8 * NT + (el >> 5), col = p.nb * 32 + (el & 31);
    float sum = s.sum[kW4Warps + w][el];
#pragma unroll
    for (int v = 1; v < kW4Warps; ++v)
      if (v > w && v <= last && ((continues >> v) & 1u)) sum = __fadd_rn(sum, s.sum[v][el]);
    if (r < s.n[p.i] && col < a.N) reinterpret_cast<uint16_t*>(a.out)[(size_t)(s.lo[p.i] + r) * a.N + col] = W4Type<DT>::round(sum);
  }
}

// NT: a unit has up to 8 NT rows; the operands of a tile are made once and multiplied NT times.
template <int DT, int SPAN, bool ZEROS, int NT>
__global__ void __launch_bounds__(kW4Threads, 1) w4_kernel(const W4Args a) {
  using Ty = W4Type<DT>;
  using St = W4Stage<SPAN, ZEROS>;
  extern __shared__ __align__(16) unsigned char s_dynamic[];  // W4Joint, then the rings [warps][kDepth][St::kBytes]
  __shared__ int s_w[kW4Warps], s_u[kW4Warps];
  W4Joint<NT>& s = *reinterpret_cast<W4Joint<NT>*>(s_dynamic);
  unsigned char* s_ring = s_dynamic + sizeof(W4Joint<NT>);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, j = lane & 3;
  const Ty ty;
  pdl_sync();

  // experts that have rows, in order, and the number of units before each (all counts are below 2^31, see the entry)
  int lo = 0, n = 0, first_row = 0, last_row = (int)a.rows;
  if (a.offsets == nullptr) {
    n = tid == 0 ? (int)a.rows : 0;
  } else {
    if (tid < a.E) {
      lo = __ldg(a.offsets + tid);
      const int hi = __ldg(a.offsets + tid + 1);
      // offsets that decrease or leave the rows are nobody's: every row becomes zero
      n = lo < 0 || hi < lo || hi > (int)a.rows ? INT_MIN : hi - lo;
    }
    first_row = __ldg(a.offsets);
    last_row = __ldg(a.offsets + a.E);
  }
  const int mine = n > 0 ? (n + 8 * NT - 1) / (8 * NT) * a.nblocks : 0;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += v;
  }
  const unsigned busy = __ballot_sync(kFull, n > 0);
  if (lane == 31) {
    s_w[warp] = __popc(busy);
    s_u[warp] = incl;
  }
  const bool broken = __syncthreads_or(n == INT_MIN);
  int at = __popc(busy & ((1u << lane) - 1u)), experts = 0, units = 0, unit_at = incl - mine;
#pragma unroll
  for (int w = 0; w < kMaxE / 32; ++w) {
    if (w < warp) {
      at += s_w[w];
      unit_at += s_u[w];
    }
    experts += s_w[w];
    units += s_u[w];
  }
  if (n > 0) {
    s.expert[at] = tid;
    s.lo[at] = lo;
    s.n[at] = n;
    s.unit[at] = unit_at;
  }
  if (broken) {
    units = 0;
    first_row = last_row = 0;
  }
  __syncthreads();

  const int even = units / gridDim.x, odd = units - even * gridDim.x;  // the first `odd` blocks have one unit more
  const int u_first = even * blockIdx.x + min((int)blockIdx.x, odd);
  const int tiles = (even + ((int)blockIdx.x < odd ? 1 : 0)) * a.chunks;
  const int t_first = (int)((int64_t)tiles * warp / kW4Warps);
  const int count = (int)((int64_t)tiles * (warp + 1) / kW4Warps) - t_first;
  W4Place here = {0, 0, 0, 0};
  if (count > 0) {
    const int ahead = t_first / a.chunks, u = u_first + ahead;
    here.c = t_first - ahead * a.chunks;
    // the last expert whose first unit is not behind u
    for (int i0 = 0;; i0 += 32) {
      const unsigned m = __ballot_sync(kFull, i0 + lane < experts && s.unit[i0 + lane] <= u);
      here.i += __popc(m);
      if (m != kFull) break;
    }
    --here.i;
    const int in = u - s.unit[here.i], passes = (s.n[here.i] + 8 * NT - 1) / (8 * NT);
    here.nb = passes == 1 ? in : in / passes;
    here.pass = in - here.nb * passes;
  }
  // to the first tile of the next unit
  auto next_unit = [&](W4Place& p) {
    p.c = 0;
    if (++p.pass * 8 * NT < s.n[p.i]) return;
    p.pass = 0;
    if (++p.nb < a.nblocks) return;
    p.nb = 0;
    ++p.i;
  };

  // copies, kDepth tiles ahead
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring) + warp * kDepth * St::kBytes;
  const unsigned char* ring_p = s_ring + warp * kDepth * St::kBytes;
  W4Place next = here;
  int to_fetch = count;
  const unsigned char *next_w = nullptr, *next_s = nullptr, *next_z = nullptr;
  auto aim = [&]() {
    const size_t block = (size_t)s.expert[next.i] * a.nblocks + next.nb;
    next_w = a.weight + (block * a.chunks + next.c) * kTileBytes + lane * 16;
    next_s = a.scales + block * a.G * 64 + g * 8;
    if (ZEROS) next_z = a.zeros + block * a.G * 16 + g * 4;
  };
  auto fetch = [&](int at_byte) {
    if (to_fetch > 0) {
      const uint32_t to = ring + at_byte;
#pragma unroll
      for (int i = 0; i < 4; ++i) copy16(to + i * 512 + lane * 16, next_w + i * 512);
      if (j < St::kParts) {
        // a group of padding alone has scale zero (its products are zero, and zero times an infinite scale is no number)
        const uint32_t of = w4_group(a, 4 * next.c + SPAN * j), gr = min(of, (uint32_t)a.G - 1);
        copy8(to + St::kScales + (j * 8 + g) * 8, next_s + (size_t)gr * 64, of == gr ? 8u : 0u);
        if (ZEROS && g < 4) copy4(to + St::kZeros + j * 16 + g * 4, next_z + (size_t)gr * 16);
      }
      next_w += kTileBytes;
      if (++next.c == a.chunks && to_fetch > 1) {
        next_unit(next);
        aim();
      }
      --to_fetch;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (count > 0) aim();
#pragma unroll 1
  for (int d = 0; d < kDepth; ++d) fetch(d * St::kBytes);

  float acc[2][NT][4];
  const unsigned char* xp[NT];
  bool began = here.c == 0;  // this warp has the unit from its first tile on
  auto begin = [&]() {
#pragma unroll
    for (int v = 0; v < NT; ++v) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[h][v][i] = 0.0f;
      // columns behind the unit's last row multiply that row again; their results are dropped
      const int row = s.lo[here.i] + min(8 * (here.pass * NT + v) + g, s.n[here.i] - 1);
      xp[v] = a.x + ((size_t)row * a.K + here.c * 128 + 8 * j) * 2;
    }
  };
  auto write = [&]() {
    const int r0 = here.pass * 8 * NT, rows = s.n[here.i] - r0, cols = a.N - here.nb * 32 - g;
    uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + (size_t)(s.lo[here.i] + r0 + 2 * j) * a.N + here.nb * 32 + g;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int v = 0; v < NT; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (8 * v + 2 * j + (i & 1) < rows && 16 * h + 8 * (i >> 1) < cols)
            o[(size_t)(8 * v + (i & 1)) * a.N + 16 * h + 8 * (i >> 1)] = Ty::round(acc[h][v][i]);
  };
  int what = 0, slot = 0;  // byte offset in the ring
  for (int t = count; t > 0;) {
    begin();
    // the rest of this unit, or of the share
    const int stretch = min(t, a.chunks - here.c);
    t -= stretch;
    const int c_end = here.c + stretch;
    // one tile with its inputs in `x`, while those of the next are fetched into `x_next` (NT = 1: more registers there
    // are not, the inputs of the other rows come from L1 when their block's turn is)
    auto tile = [&](const uint4 (&x)[4], uint4 (&x_next)[4]) {
      if (NT == 1) {
        xp[0] += 256;
        if (here.c + 1 < c_end) w4_load_x(a, xp[0], here.c + 1, x_next);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();  // the scales of a tile are copied by all lanes
      const unsigned char* st = ring_p + slot;
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(st + i * 512 + lane * 16);
      uint2 sc[St::kParts];
      uint32_t zp[St::kParts];
#pragma unroll
      for (int k = 0; k < St::kParts; ++k) {
        sc[k] = *reinterpret_cast<const uint2*>(st + St::kScales + (k * 8 + g) * 8);
        zp[k] = ZEROS ? *reinterpret_cast<const uint16_t*>(st + St::kZeros + k * 16 + g * 2) : 0x8888u;
      }
      __syncwarp();
      fetch(slot);
      slot = slot + St::kBytes == kDepth * St::kBytes ? 0 : slot + St::kBytes;
      w4_tile<DT, SPAN, NT>(
          ty, w, [&](int q, int v) { return NT == 1 ? x[q] : w4_load_x(a, xp[v], here.c, q); },
          [&](int k, int i) {
            const uint32_t v = i < 2 ? sc[k].x : sc[k].y;
            return i & 1 ? Ty::second(v) : Ty::first(v);
          },
          [&](int k, int i) { return Ty::zero_operand((zp[k] >> (4 * i)) & 15u); }, acc);
      if (NT > 1) {
#pragma unroll
        for (int v = 0; v < NT; ++v) xp[v] += 256;
      }
      ++here.c;
    };
    uint4 x0[4], x1[4];
    if (NT == 1) w4_load_x(a, xp[0], here.c, x0);
#pragma unroll 1
    while (true) {
      tile(x0, x1);
      if (here.c == c_end) break;
      if (NT > 1) continue;
      tile(x1, x0);
      if (here.c == c_end) break;
    }
    const bool ended = here.c == a.chunks;
    if (began && ended) {
      write();
    } else {
      float* to = s.sum[began ? kW4Warps + warp : warp];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < NT; ++v)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[(8 * v + 2 * j + (i & 1)) * 32 + 16 * h + 8 * (i >> 1) + g] = acc[h][v][i];
      what |= began ? kBegins : ended ? kContinues | kEnds : kContinues;
    }
    if (t > 0) {
      next_unit(here);
      began = true;
    }
  }
  if (lane == 0) {
    s.what[warp] = what;
    s.place[warp] = here;
  }
  __syncthreads();
  w4_join<DT, NT>(a, s);

  // rows of no expert
  const int64_t before = (int64_t)first_row * a.N, idle = before + (a.rows - last_row) * a.N;
  for (int64_t k = (int64_t)blockIdx.x * kW4Threads + tid; k < idle; k += (int64_t)gridDim.x * kW4Threads)
    reinterpret_cast<uint16_t*>(a.out)[k < before ? k : (int64_t)last_row * a.N + (k - before)] = 0;
}

// The layout of the weights, once when a program loads them: a thread makes one 16-byte vector (four words) of a tile.
__global__ void __launch_bounds__(256) pack_w4_kernel(const unsigned char* __restrict__ q, uint4* __restrict__ out, int64_t vectors, int N,
                                                      int half, int blocks, int chunks) {
  pdl_sync();
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < vectors; v += (int64_t)gridDim.x * 256) {
    const int lane = (int)(v & 31), part = (int)(v >> 5) & 3;
    const int64_t tile = v >> 7, eb = tile / chunks, e = eb / blocks;
    const int c = (int)(tile - eb * chunks), n = (int)(eb - e * blocks) * 32 + part * 8 + (lane >> 2);
    const unsigned char* row = q + ((size_t)e * N + n) * half;
    uint32_t o[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int at = 64 * c + 16 * m + 4 * (lane & 3);
      const uint32_t w = n < N && at < half ? __ldg(reinterpret_cast<const uint32_t*>(row + at)) : 0u;
      o[m] = 0u;
#pragma unroll
      for (int p = 0; p < 4; ++p) o[m] |= ((w >> (8 * p)) & 15u) << (4 * p) | ((w >> (8 * p + 4)) & 15u) << (16 + 4 * p);
    }
    out[v] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int DT, int SPAN, bool ZEROS, int NT>
cudaError_t launch_w4(const W4Args& a, cudaStream_t s) {
  constexpr int smem = sizeof(W4Joint<NT>) + kW4Warps * kDepth * W4Stage<SPAN, ZEROS>::kBytes;
  static_assert(sizeof(W4Joint<NT>) % 16 == 0, "the rings are 16-byte aligned");
  static std::atomic<uint64_t> set{0};  // devices whose kernel has its shared memory; setting it twice does no harm
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!((set.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(w4_kernel<DT, SPAN, ZEROS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    set.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  }
  return launch_pdl(w4_kernel<DT, SPAN, ZEROS, NT>, dim3((unsigned)device_sms()), dim3(kW4Threads), smem, s, a);
}

template <int DT, int SPAN, bool ZEROS>
cudaError_t launch_w4_rows(const W4Args& a, cudaStream_t s) {
  // 8 experts x 8192 outputs x 7168 inputs, units of 8 / of 16 rows: 1 row each 49 / 51 us, 8 rows 52 / 72, 9 rows 93 / 73,
  // 16 rows 96 / 75, 32 rows 193 / 165.  The host knows the rows of all experts together, not of each: units of 16 where
  // an expert has more than 8 on average.
  return a.rows > 8 * (int64_t)a.E ? launch_w4<DT, SPAN, ZEROS, 2>(a, s) : launch_w4<DT, SPAN, ZEROS, 1>(a, s);
}

template <int DT, bool ZEROS>
cudaError_t launch_w4_span(const W4Args& a, int group, cudaStream_t s) {
  if (group % 128 == 0) return launch_w4_rows<DT, 4, ZEROS>(a, s);
  if (group % 64 == 0) return launch_w4_rows<DT, 2, ZEROS>(a, s);
  return launch_w4_rows<DT, 1, ZEROS>(a, s);
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_pack_w4(int32_t E, int32_t N, int32_t K, const uint8_t* q, void* weight, void* stream) {
  if (E < 1 || E > kMaxE || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 20) || K % 32 != 0) return MOE_RD_E_SHAPE;
  if (q == nullptr || weight == nullptr) return MOE_RD_E_NULL;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(weight)) & 15) return MOE_RD_E_ALIGN;
  const int blocks = (N + 31) / 32, chunks = (K + 127) / 128;
  const int64_t vectors = (int64_t)E * blocks * chunks * (kTileBytes / 16);
  const int64_t want = (vectors + 255) / 256, cap = (int64_t)device_sms() * 64;
  const cudaError_t e = launch_pdl(pack_w4_kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, static_cast<cudaStream_t>(stream),
                                   static_cast<const unsigned char*>(q), static_cast<uint4*>(weight), vectors, (int)N, K / 2, blocks, chunks);
  count_launch();
  if (e != cudaSuccess) set_last_cuda_error(e);
  return e == cudaSuccess ? MOE_RD_OK : MOE_RD_E_CUDA;
}

extern "C" int moe_rd_expert_matvec_w4(int64_t rows, int32_t N, int32_t K, int32_t E, int32_t group, int32_t dtype,
                                       const void* x, const void* weight, const void* scales, const uint16_t* zeros,
                                       const int32_t* offsets, void* out, void* stream) {
  if (dtype == MOE_RD_T_F32) return MOE_RD_E_UNSUPPORTED;
  if (dtype != MOE_RD_T_BF16 && dtype != MOE_RD_T_FP16) return MOE_RD_E_ENUM;
  if (rows < 0 || rows > (1 << 30) || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 20) || E < 1 || E > kMaxE ||
      group < 32 || group % 32 != 0 || K % group != 0 || (offsets == nullptr && E != 1))
    return MOE_RD_E_SHAPE;
  // tiles are counted in 32 bits
  if ((rows / 8 + E) * ((N + 31) / 32) > 0x7fffffff / ((K + 127) / 128)) return MOE_RD_E_TOO_LARGE;
  if (rows == 0) return MOE_RD_OK;
  if (x == nullptr || weight == nullptr || scales == nullptr || out == nullptr) return MOE_RD_E_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(scales) |
       reinterpret_cast<uintptr_t>(zeros)) & 15 ||
      reinterpret_cast<uintptr_t>(out) & 1)
    return MOE_RD_E_ALIGN;
  W4Args a = {};
  a.x = static_cast<const unsigned char*>(x);
  a.weight = static_cast<const unsigned char*>(weight);
  a.scales = static_cast<const unsigned char*>(scales);
  a.zeros = reinterpret_cast<const unsigned char*>(zeros);
  a.offsets = offsets;
  a.out = static_cast<unsigned char*>(out);
  a.rows = rows;
  a.N = N;
  a.K = K;
  a.E = E;
  a.G = K / group;
  a.chunks = (K + 127) / 128;
  a.nblocks = (N + 31) / 32;
  const uint32_t per = (uint32_t)group / 32;
  a.group_magic = per == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + per - 1) / per);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == MOE_RD_T_BF16)
    e = zeros != nullptr ? launch_w4_span<MOE_RD_T_BF16, true>(a, group, s) : launch_w4_span<MOE_RD_T_BF16, false>(a, group, s);
  else
    e = zeros != nullptr ? launch_w4_span<MOE_RD_T_FP16, true>(a, group, s) : launch_w4_span<MOE_RD_T_FP16, false>(a, group, s);
  count_launch();
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return MOE_RD_E_CUDA;
  }
  return MOE_RD_OK;
}
