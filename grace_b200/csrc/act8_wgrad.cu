// Weight gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//   dW[n, k] = sum_m dY[m, n] x~[m, k]      db[n] = sum_m dY[m, n]
// without ever writing x~ to memory: its tiles are decoded on the way into the tensor core.
//
// A pair of CTAs computes a dW^T tile of 256 input features by 256 output features, D[k, n] += A[k, m] B[m, n], in steps of
// 64 tokens (tcgen05.mma with cta_group::2: each CTA holds 128 rows of A, 128 columns of B, and the accumulator rows
// that belong to its part of A).  Both operands have the tokens as their contracted axis and lie in memory with the
// OTHER axis contiguous, which the tensor core takes as it is (MN-major operands, 128-byte rows of 64 elements in the
// 128-byte swizzle), so nothing is transposed:
//   B = dY     TMA boxes of 64 tokens x 64 output features land in the operand layout
//   A = x~     TMA brings the codes (64 tokens x 128 bytes), the decoders fetch their scale bytes; three groups of four warps take the steps in turn, decode them
//              and store the operand tile
// For bf16 a code's low seven bits are placed under an exponent that already holds the scale, its sign bit under
// another, so decoding and scaling are one subtraction of two bf16 pairs; the result is exact.  (fp16: see decode8.)
//
// Roles: warp 0 loads dY, warp 2 the codes (both by TMA), warp 1 of the pair's first CTA issues the MMAs, warp 3 adds up
// the bias gradient (the CTAs of a row of tiles share its columns), warps 4 - 15 decode, warps 16 - 19 write results
// from one of two accumulators while the MMAs fill the other.  dY waits in seven stages, the codes in five, the decoded
// operand in four: a step is on its way for about seven steps' time (load 950 cycles, decode 1100, MMA 512, barriers
// between), but only its dY is needed all that long.
//
// A pair takes whole tiles, one from each full wave of them, so that neighbouring pairs read the same rows at the same
// time.  The tiles of the last, partial wave are laid end to end and cut into equal runs of steps, one for each pair
// (where that saves more than it costs: see make_plan); a run that is not a whole tile leaves fp32 partial sums
// in a workspace, and a second kernel adds a tile's runs in order (no atomics: the same bits on every run).
//
// The tensor core truncates where it adds to an fp32 accumulator, which adds up to a bias that grows with the tokens (2.2e-6
// of the result after 4096 of them, half a step of fp16 after some hundred thousand).  The accumulator is therefore emptied every 1536
// tokens for an fp32 result and every 2048 for a 16-bit one into the other accumulator's place, rounding to nearest; kept in
// the output instead, that cost 40 % more traffic through L2 and as much time.  What is left of the bias (some 1e-6) does not
// grow any more.  Sums are fp32 throughout, rounded once to the output's type.
//
// What bounds it: in a large product, shared memory. A step moves 96 KB in and out of an SM's (dY and codes in, codes out and
// operand in for the decoders, both operands out for the product), 750 cycles at its 128 bytes a cycle, where the product
// itself takes 512; a step takes 800 to 860, and emptying the accumulator, when the products stop, 8 % on top of that.  Measured
// with cold caches: 16384 tokens, 4096 x 4096, bf16 430 us (1279 TFLOP/s, 0.80 of the measured library rate; the library's product
// of two bf16 matrices takes 336), fp16 470, fp32 result 453 us.  A call of less than a wave of tiles takes longer a step: 4096
// tokens, 4096 x 1024, fp32 result 50 us, 1500 cycles for each of its 64 steps (64 tiles for 74 pairs, library 31); the
// accumulator is emptied three times in them, which explains a part of it, and the rest has not been found.  1024 x 1024 with its
// bias 19 + 9 us (library 16): runs of 14 steps, and a second kernel for their sums.  One warp adds up the bias columns: free where
// many tiles along the inputs share them, not where few do (16384 tokens, 4096 outputs, without and with it: 128 inputs 45 and 77
// us, 512 inputs 71 and 98, 1024 inputs 128 and 147, 4096 inputs 430 and 439).
//
// Every wait is bounded; when one runs out the status block says which and the outputs are NaN.
#include <type_traits>

#include "act8.cuh"
#include "act8.h"
#include "gradio.cuh"
#include "tensor_core.cuh"

namespace grace {
namespace {

constexpr int kThreads = 640;
constexpr int kTileK = 128;            // input features of a CTA's half of the tile
constexpr int kTileN = 256;            // output features of a tile
constexpr int kHalfN = 128;            // of them in one CTA's shared memory
constexpr int kStep = 64;              // tokens of a step
constexpr int kBoxBytes = kStep * 128; // 64 tokens x 64 features of 16 bits
constexpr int kBStages = 7, kCodeStages = 5, kAStages = 4;
constexpr int kDecodeWarp0 = 4, kGroups = 3, kGroupWarps = 4, kEpilogueWarp0 = kDecodeWarp0 + kGroups * kGroupWarps;
constexpr int kMinSavedSteps = 24;
// Steps between two emptyings of the accumulator, fp32 and 16-bit results (see the header).  4096 x 4096 at 16384 tokens: an fp32
// result takes 435 us and is off by 2.2e-6 with 64 steps, 453 and 0.6e-6 with 24, 487 and 0.3e-6 with 12; a bf16 one 409 us never
// emptied, 420 with 64 steps, 434 with 32, 442 with 24, and differs from the rounded product of fp32 matrices by 21e-5, 9.8e-5,
// 8.0e-5 and 7.7e-5 of itself, of which 7.4e-5 are that product's.
constexpr int kChunkStepsF32 = 24, kChunkSteps16 = 32;
constexpr unsigned long long kTimeoutNs = 2000000000ull;
constexpr unsigned kTmemCols = 512;

struct __align__(1024) WgradSmem {
  unsigned char b[kBStages][2 * kBoxBytes];
  unsigned char a[kAStages][2 * kBoxBytes];
  unsigned char codes[kCodeStages][kStep * kTileK];
  unsigned long long b_full[kBStages];                             // dY has landed
  unsigned long long b_used[kBStages], b_summed[kBStages];         // the MMAs, the bias warp are done with it
  unsigned long long c_full[kCodeStages], c_empty[kCodeStages];    // the codes have landed, are in registers
  unsigned long long ready[kAStages];                              // first CTA of the pair: both CTAs' operands are in place
  unsigned long long acc_full[2], acc_empty[2];                    // (acc_empty: first CTA)
  unsigned long long done;
  unsigned tmem_base;
  unsigned failed;                                                 // a wait of this CTA ran out
  int rest[2][4];                                                  // this pair's pieces of the last wave (a Piece each; st1 = 0: none)
};
static_assert(sizeof(WgradSmem) + 1024 <= 227 * 1024, "shared memory");
static_assert(kAStages <= kCodeStages && kAStages <= kBStages, "see the decoders' waits");

constexpr int kPartFloats = 2 * kTileN * kTileK;    // partial sums of a tile: [2 CTAs][256][128]
constexpr int kSlotFloats = kPartFloats + 2 * kHalfN;   // and of its CTAs' bias columns

struct WgradArgs {
  const unsigned char* scales;
  int spitch;
  long long tokens;
  int outs, ins;        // N, K
  int tiles_k;          // pair tiles along the input features
  int pairs;            // of CTAs
  int whole;            // whole tiles a pair takes: tiles pair, pair + pairs, ...
  int rest, rest_pairs; // tiles after them, and the pairs that share their steps equally
  int steps;            // of 64 tokens, over all tokens
  int chunk;            // steps between two emptyings of the accumulator
  int single;           // 1: a piece may take several emptyings, which are added up in the second accumulator's place
  unsigned one;         // 1 (see decode8)
  int bias_cols;        // columns of its 128 that a CTA adds up (a power of two, 8 to 128), 0: no bias gradient
  void* out;
  void* bias;
  float* work;          // [2 * rest_pairs][kSlotFloats]: runs that are not whole tiles
};

// A piece of work of a pair: steps [st0, st1) of a tile.
struct Piece {
  int tile, st0, st1;
  int slot;             // of the workspace; -1: a whole tile, straight to the output
};
// A pair's run of the last wave is no longer than a tile, so it touches two tiles at most: j = 0 or 1.
__device__ __forceinline__ Piece rest_piece(const WgradArgs& a, int pair, int j) {
  Piece p{0, 0, 0, -1};
  if (pair >= a.rest_pairs) return p;
  const long long total = (long long)a.rest * a.steps;
  const long long lo = pair * total / a.rest_pairs, hi = (pair + 1) * total / a.rest_pairs;
  const int r = (int)(lo / a.steps) + j;
  p.st0 = j ? 0 : (int)(lo - (long long)r * a.steps);
  p.st1 = (int)max(0ll, min((long long)a.steps, hi - (long long)r * a.steps));
  p.tile = a.whole * a.pairs + r;
  p.slot = p.st0 == 0 && p.st1 == a.steps ? -1 : pair * 2 + j;
  return p;
}
__device__ __forceinline__ bool piece_at(const WgradArgs& a, const WgradSmem& sm, int pair, int i, Piece& p) {
  if (i < a.whole) {
    p = {pair + i * a.pairs, 0, a.steps, -1};
    return true;
  }
  i -= a.whole;   // (whole warps call this: what it reads is made uniform)
  if (i > 1 || __shfl_sync(0xffffffffu, sm.rest[i][2], 0) == 0) return false;
  p = {__shfl_sync(0xffffffffu, sm.rest[i][0], 0), __shfl_sync(0xffffffffu, sm.rest[i][1], 0), __shfl_sync(0xffffffffu, sm.rest[i][2], 0),
       __shfl_sync(0xffffffffu, sm.rest[i][3], 0)};
  return true;
}

// The status block of the bounded waits (common.cuh), one for each device, sticky until act8_wgrad_status clears it.  A
// symbol and not an allocation, so that the first call may be made while a graph is being captured.
__device__ unsigned wgrad_status[16];

__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"((unsigned)accum) : "memory");
}
// Arrives at the barrier of the same name in both CTAs of the pair when the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(void* bar, unsigned ctas) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"((unsigned short)ctas)
               : "memory");
}
// Arrives at the barrier of the same name in another CTA (`cta`: rank in the cluster).  What the barrier announces is
// this CTA's own operand tile, which its threads have handed to the async proxy by a fence of their own; nothing is
// read from here through the generic proxy.  The arrival therefore needs no cluster-wide release, which (with the
// acquire on the other side) took 1300 cycles each, more than two steps of the tensor core.
__device__ __forceinline__ void mbar_arrive_at(void* bar, unsigned cta) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(bar)), "r"(cta));
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Eight codes as a 16-byte operand chunk.  The codes of a word come out as its even bytes, then its odd bytes, which one
// mask each finds in place: input features 1 and 2 of every four change places in the operand, and so do the lanes of
// the result (feature_of).  Integer operations have half the rate of the others and bound this kernel's decoders; `one` is
// 1, and multiplying by it puts an addition into the multipliers' pipe.
__device__ __forceinline__ int feature_of(int lane) { return (lane & ~3) | ((lane & 1) << 1) | ((lane >> 1) & 1); }

__device__ __forceinline__ uint4 decode8(uint2 c, unsigned s, unsigned one, __nv_bfloat16) {
  // exponent field s + 7: 2^(s - 127) * 128 * (1 + m / 128) = (128 + m) steps
  const unsigned base = s == 255u ? 0x7fc07fc0u : ((s + 7u) << 7) * 0x10001u;
  const unsigned w[4] = {c.x, c.x >> 8, c.y, c.y >> 8};
  unsigned r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned hi = (w[j] & 0x007f007fu) | base;             // (128 + low seven bits) steps
    const unsigned lo = (w[j] & 0x00800080u) * one + base;       // 128 steps, or 256 for a negative code
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&hi), *reinterpret_cast<const __nv_bfloat162*>(&lo));
    r[j] = *reinterpret_cast<const unsigned*>(&d);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// fp16 has the significand to take a code whole (1024 + byte), but not the exponents: the scale goes on in two factors,
// 2^-6 and 2^(s - 121), so that its range reaches from 2^-30 to 2^9, that of groups of fp16 values (2^-7 and 2^-24 for one
// scale more, which only groups of wider types have); the first product is exact and the second rounds once, into the
// subnormals.  A group with a value of 2^16 or more reads as NaN.
__device__ __forceinline__ uint4 decode8(uint2 c, unsigned s, unsigned, __half) {
  // 2^(s - 121): normal or subnormal; below s = 96 every value is below 2^-25 and rounds to zero
  const bool least = s == 96u;
  const unsigned f = s > 136u ? 0x7e00u : (s >= 107u ? (s - 106u) << 10 : (s >= 97u ? 1u << (s - 97u) : (least ? 1u : 0u)));
  const __half2 scale = __half2half2(__ushort_as_half((unsigned short)f));
  const __half2 sixth = __half2half2(__ushort_as_half(least ? 0x2000 : 0x2400));       // 2^-6, or 2^-7,
  const __half2 offset = __half2half2(__ushort_as_half(least ? 0xc880 : 0xcc80));      // times -1152: -18, or -9
  c.x ^= 0x80808080u;
  c.y ^= 0x80808080u;
  const unsigned w[4] = {c.x, c.x >> 8, c.y, c.y >> 8};
  unsigned r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned v = (w[j] & 0x00ff00ffu) | 0x64006400u;   // 1024 + code + 128
    const __half2 d = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&v), sixth, offset), scale);
    r[j] = *reinterpret_cast<const unsigned*>(&d);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// fp32 accumulator, both operands T and MN-major, M = 256; N is added at run time
template <class T> constexpr uint32_t instruction_desc() {
  constexpr uint32_t f = __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(2 * kTileK >> 4) << 24);
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
        "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
        "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]), "r"(addr) : "memory");
}
// (the registers are operands so that nothing that uses them can be moved before the wait)
__device__ __forceinline__ void tmem_wait_load(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                 "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :: "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Lane l holds v[0 .. 7] of row l of a 32 x 8 block: afterwards w is eight neighbouring rows, (l & 24) .. (l & 24) + 7, of column
// l & 7, rounded to the 16-bit type O: 16 bytes of an output row instead of two of eight of them.
template <class O>
__device__ __forceinline__ uint4 turn8(const float* v, int lane) {
  unsigned p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool odd = lane & 1;
    const float other = __shfl_xor_sync(0xffffffffu, odd ? v[2 * j] : v[2 * j + 1], 1);
    p[j] = odd ? pack2<O>(other, v[2 * j + 1]) : pack2<O>(v[2 * j], other);
  }
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & b) continue;
      const bool up = lane & (2 * b);
      const unsigned other = __shfl_xor_sync(0xffffffffu, up ? p[j] : p[j | b], 2 * b);
      if (up) p[j] = other;
      else p[j | b] = other;
    }
  // (features 1 and 2 of every four back in their places: see decode8)
  return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x5410),
                    __byte_perm(p[2], p[3], 0x7632));
}

// A tile as one of the pair's CTAs sees it.
struct Tile {
  int k0;        // its first input feature
  int n0;        // the tile's first output feature
  int boxes;     // 64-feature boxes of B in each of the two CTAs
  int share;     // which share of the bias columns this row of tiles' CTA adds up
};
__device__ __forceinline__ Tile tile_at(const WgradArgs& a, int tile, int half) {
  const int tk = tile % a.tiles_k, tn = tile / a.tiles_k;
  return {(tk * 2 + half) * kTileK, tn * kTileN, a.outs - tn * kTileN > 2 * 64 ? 2 : 1, tk};
}

// One lane of a converged warp.  The roles that issue TMA loads and MMAs run as whole warps and elect a lane only around
// the instruction: descriptors and coordinates then stay in uniform registers, where the instruction wants them.  As a
// single diverged lane, issuing a step took longer than the tensor core took to compute it.
__device__ __forceinline__ bool elect_one() {
  unsigned one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// A ring position and the parity of its use.
template <int N> struct Ring {
  unsigned slot = 0, parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) { slot = 0; parity ^= 1; }
  }
};
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <class T, class O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_codes, const WgradArgs a) {
  extern __shared__ unsigned char raw[];
  WgradSmem& sm = *reinterpret_cast<WgradSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const Status status{wgrad_status};
  const int half = blockIdx.x & 1, pair = blockIdx.x >> 1;
  const bool has_bias = a.bias_cols != 0;
  const unsigned two = a.single ? 0u : 1u;       // accumulators less one
  Piece p;
  cudaTriggerProgrammaticLaunchCompletion();     // (the second kernel's blocks take an SM as soon as one is left; it waits for all)

  if (warp == 0) {      // (a lane for each stage)
    if (lane < kBStages) { mbar_init(&sm.b_full[lane], 1); mbar_init(&sm.b_used[lane], 1); mbar_init(&sm.b_summed[lane], 1); }
    if (lane < kCodeStages) { mbar_init(&sm.c_full[lane], 1); mbar_init(&sm.c_empty[lane], kGroupWarps); }
    if (lane < kAStages) mbar_init(&sm.ready[lane], 2 * kGroupWarps);
    if (lane < 2) { mbar_init(&sm.acc_full[lane], 1); mbar_init(&sm.acc_empty[lane], 2 * 4); }
    if (lane == 0) { mbar_init(&sm.done, 1); sm.failed = 0; }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32 * 3) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_dy) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_codes) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 2 && lane < 2) {
    p = rest_piece(a, pair, lane);
    sm.rest[lane][0] = p.tile;
    sm.rest[lane][1] = p.st0;
    sm.rest[lane][2] = p.st1;
    sm.rest[lane][3] = p.slot;
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ---- dY ----
    bool ok = true;
    unsigned it = 0;
    Ring<kBStages> r;
    for (int i = 0; ok && piece_at(a, sm, pair, i, p); ++i) {
      const Tile t = tile_at(a, p.tile, half);
      for (int st = p.st0; st < p.st1; ++st, ++it, r.next()) {
        if (it >= kBStages) {
          ok = mbar_wait_hint(&sm.b_used[r.slot], r.parity ^ 1, kTimeoutNs, status, 100 + r.slot) &&
               (!has_bias || mbar_wait_hint(&sm.b_summed[r.slot], r.parity ^ 1, kTimeoutNs, status, 150 + r.slot));
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (elect_one()) {
          mbar_expect_tx(&sm.b_full[r.slot], t.boxes * kBoxBytes);
          for (int j = 0; j < t.boxes; ++j)
            tma_load_2d(sm.b[r.slot] + j * kBoxBytes, &map_dy, t.n0 + (half * t.boxes + j) * 64, st * kStep, &sm.b_full[r.slot]);
        }
        __syncwarp();
      }
    }
    // At the end the last arrivals of the pair's MMAs must have landed here (see the MMAs); where a consumer gave up, the
    // loads that were issued, before the shared memory is let go.
    bool landed = true;
    for (unsigned s = it > kBStages ? it - kBStages : 0; s < it; ++s)
      landed = mbar_wait_hint(ok ? &sm.b_used[s % kBStages] : &sm.b_full[s % kBStages], (s / kBStages) & 1, 2 * kTimeoutNs, status, 400) && landed;
    landed = mbar_wait_hint(&sm.done, 0, 2 * kTimeoutNs, status, 800) && landed;
    if (!ok || !landed) sm.failed = 1;
  } else if (warp == 1) {
    // ---- MMAs, by one thread of the pair ----
    if (half == 0) {
      // (addresses in a descriptor are in units of 16 bytes, in its low bits)
      const uint64_t a_desc = smem_desc(smem_u32(sm.a), kBoxBytes, 1024, 2), b_desc = smem_desc(smem_u32(sm.b), kBoxBytes, 1024, 2);
      unsigned item = 0;
      Ring<kAStages> ra;
      Ring<kBStages> rb;
      bool ok = true;
      for (int i = 0; ok && piece_at(a, sm, pair, i, p); ++i) {
        const Tile t = tile_at(a, p.tile, 0);
        const uint32_t idesc = instruction_desc<T>() | ((uint32_t)(t.boxes * 128 >> 3) << 17);
        for (int st = p.st0; ok && st < p.st1; ++item) {
          const unsigned buf = item & two, use = item >> two;
          if (use >= 1) ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.acc_empty[buf], (use - 1) & 1, kTimeoutNs, status, 300 + buf));
          if (!ok) break;
          tc_fence_after();
          const int end = min(st + a.chunk, p.st1);
          for (bool fresh = true; st < end; ++st, ra.next(), rb.next(), fresh = false) {
            ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.ready[ra.slot], ra.parity, kTimeoutNs, status, 200 + ra.slot));
            if (!ok) break;
            tc_fence_after();
            const uint64_t ad = a_desc + ra.slot * (2 * kBoxBytes >> 4), bd = b_desc + rb.slot * (2 * kBoxBytes >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kStep / 16; ++kk)   // 16 tokens: two groups of eight 128-byte rows; the next 64 features one box further
                umma_f16_pair(tmem + buf * kTileN, ad + kk * (2048 >> 4), bd + kk * (2048 >> 4), idesc, kk > 0 || !fresh);
              umma_commit_pair(&sm.b_used[rb.slot], 3u);
            }
            __syncwarp();
          }
          if (ok && elect_one()) umma_commit_pair(&sm.acc_full[buf], 3u);
          __syncwarp();
        }
      }
      if (elect_one()) umma_commit_pair(&sm.done, 3u);
      __syncwarp();
      // The other CTA's last arrivals here are on their way without being waited for by anything else, and a barrier
      // between the CTAs does not order them: this CTA has to be there when they land.
      for (unsigned n = item > two + 1 ? item - two - 1 : 0; ok && n < item; ++n)
        ok = mbar_wait_hint(&sm.acc_empty[n & two], (n >> two) & 1, 2 * kTimeoutNs, status, 350);
      if (!ok) sm.failed = 1;
    }
  } else if (warp == 2) {
    // ---- codes ----
    bool ok = true;
    unsigned it = 0;
    Ring<kCodeStages> r;
    for (int i = 0; ok && piece_at(a, sm, pair, i, p); ++i) {
      const Tile t = tile_at(a, p.tile, half);
      for (int st = p.st0; st < p.st1; ++st, ++it, r.next()) {
        if (it >= kCodeStages) ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.c_empty[r.slot], r.parity ^ 1, kTimeoutNs, status, 500 + r.slot));
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&sm.c_full[r.slot], kStep * kTileK);
          tma_load_2d(sm.codes[r.slot], &map_codes, t.k0, st * kStep, &sm.c_full[r.slot]);
        }
        __syncwarp();
      }
    }
    if (!ok)
      for (unsigned s = it > kCodeStages ? it - kCodeStages : 0; s < it; ++s) mbar_wait_hint(&sm.c_full[s % kCodeStages], (s / kCodeStages) & 1, kTimeoutNs, status, 450);
  } else if (warp == 3) {
    // ---- bias gradient: this CTA's share of its columns, eight a thread, the step's tokens dealt to the threads ----
    if (has_bias) {
      const int chunks = a.bias_cols >> 3;                     // 1 .. 16 chunks of eight columns
      const int sub = lane / chunks, rows = 32 / chunks;       // a thread takes the tokens sub, sub + rows, ...
      unsigned it = 0;
      bool ok = true;
      for (int i = 0; piece_at(a, sm, pair, i, p); ++i) {        // (after a failure too: all that is left of the bias is NaN)
        const Tile t = tile_at(a, p.tile, half);
        const int col = t.share * a.bias_cols + (lane % chunks) * 8;      // (tiles past the last share have none)
        const bool mine = col < t.boxes * 64;
        float acc[8] = {};
        for (int st = p.st0; ok && st < p.st1; ++st, ++it) {
          const unsigned slot = it % kBStages;
          ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.b_full[slot], (it / kBStages) & 1, kTimeoutNs, status, 550 + slot));
          if (!ok) break;
          if (mine) {
            const unsigned char* q = sm.b[slot] + (col >> 6) * kBoxBytes;
            const int c = (col >> 3) & 7;
#pragma unroll 4
            for (int m = sub; m < kStep; m += rows) {
              Chunk8<T> x;
              x.w = *reinterpret_cast<const uint4*>(q + m * 128 + ((c ^ (m & 7)) << 4));
              float v[8];
              x.get(v);
#pragma unroll
              for (int j = 0; j < 8; ++j) acc[j] += v[j];
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.b_summed[slot]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int o = chunks; o < 32; o <<= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
        if (lane < chunks && mine) {
          const int n = t.n0 + half * t.boxes * 64 + col;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = ok ? acc[j] : __uint_as_float(0x7fffffffu);
            if (p.slot >= 0) a.work[(size_t)p.slot * kSlotFloats + kPartFloats + half * kHalfN + col + j] = x;
            else if (n + j < a.outs) static_cast<O*>(a.bias)[n + j] = from_f32<O>(x);
          }
        }
      }
    }
  } else if (warp < kEpilogueWarp0) {
    // ---- decode: a thread takes sixteen codes (two 16-byte operand chunks) of four tokens a step ----
    const unsigned group = (warp - kDecodeWarp0) / kGroupWarps;
    const int t = (tid - kDecodeWarp0 * 32) & (kGroupWarps * 32 - 1);
    const int c = t & 7, row0 = t >> 3, swap = c >> 2;      // eight threads of a row hit eight different 16-byte banks each time
    const int j0 = (c & 3) * 2 + swap, j1 = (c & 3) * 2 + 1 - swap;
    unsigned it = 0, sc[4];
    // the scale bytes of a step's four tokens, asked for one of the group's steps (three in all) ahead
    auto scales_of = [&](const Tile& tile, int st) {
      const int at = (tile.k0 >> 5) + (c >> 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long row = (long long)st * kStep + row0 + 16 * j;
        sc[j] = row < a.tokens && at < a.spitch ? __ldg(a.scales + row * a.spitch + at) : 0u;    // past the end: zeros
      }
    };
    bool ok = true;
    for (int i = 0; ok && piece_at(a, sm, pair, i, p); ++i) {
      const Tile tile = tile_at(a, p.tile, half);
      int st = p.st0 + (int)((group + kGroups - it % kGroups) % kGroups);     // the group's first step of this piece
      const unsigned it0 = it - p.st0;
      if (st < p.st1) scales_of(tile, st);
      for (; st < p.st1; st += kGroups) {
        const unsigned n = it0 + st, cs = n % kCodeStages, as = n % kAStages;      // n: steps before this one
        // The operand slot is free when the MMAs of the step that had it are done.  This wait comes before the one for the
        // codes, and not only for that: a parity tells a phase from its neighbours alone, loads may land out of order, and a
        // group does not look at the other groups' steps.  That an MMA is done means that the codes of all steps before it
        // have been decoded, so that the codes' barrier is in this step's phase or past it.
        if (n >= kAStages) ok = mbar_wait_hint(&sm.b_used[(n - kAStages) % kBStages], ((n - kAStages) / kBStages) & 1, kTimeoutNs, status, 620 + as);
        if (ok) ok = mbar_wait_hint(&sm.c_full[cs], (n / kCodeStages) & 1, kTimeoutNs, status, 600 + cs);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        uint4 q[4];
        unsigned s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[j] = *reinterpret_cast<const uint4*>(&sm.codes[cs][(row0 + 16 * j) * kTileK + c * 16]);
          s[j] = sc[j];
        }
        if (st + kGroups < p.st1) scales_of(tile, st + kGroups);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.c_empty[cs]);   // (the warp's codes are in registers)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = row0 + 16 * j;
          unsigned char* const row = sm.a[as] + swap * kBoxBytes + m * 128;
          const uint2 u = swap ? make_uint2(q[j].z, q[j].w) : make_uint2(q[j].x, q[j].y);
          const uint2 v = swap ? make_uint2(q[j].x, q[j].y) : make_uint2(q[j].z, q[j].w);
          *reinterpret_cast<uint4*>(row + ((j0 ^ (m & 7)) << 4)) = decode8(u, s[j], a.one, T{});
          *reinterpret_cast<uint4*>(row + ((j1 ^ (m & 7)) << 4)) = decode8(v, s[j], a.one, T{});
        }
        fence_async_shared();   // the tensor core reads the tile through the async proxy
        ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.b_full[n % kBStages], (n / kBStages) & 1, kTimeoutNs, status, 640));   // the step's dY is here too
        if (!ok) break;
        __syncwarp();      // (lane 0 arrives for the whole warp's stores; a vote orders no memory)
        if (lane == 0) mbar_arrive_at(&sm.ready[as], 0);
      }
      it += p.st1 - p.st0;
    }
    if (!ok) sm.failed = 1;
  } else {
    // ---- results: TMEM lane = input feature, column = output feature ----
    const int kl = (warp - kEpilogueWarp0) * 32 + feature_of(lane);
    unsigned item = 0;
    bool ok = true;
    for (int i = 0; piece_at(a, sm, pair, i, p); ++i) {
      const Tile t = tile_at(a, p.tile, half);
      const int k = t.k0 + kl, cols = t.boxes * 128;
      const uint32_t quarter = (uint32_t)((warp - kEpilogueWarp0) * 32) << 16;
      for (int st = p.st0; st < p.st1; st += a.chunk, ++item) {
        const unsigned buf = item & two, use = item >> two;
        const bool add = st > p.st0, last = st + a.chunk >= p.st1;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_hint(&sm.acc_full[buf], use & 1, 2 * kTimeoutNs, status, 700 + buf));
        tc_fence_after();
        const uint32_t base = tmem + buf * kTileN + quarter, sums = tmem + kTileN + quarter;
        // columns c .. c + 31 of the accumulator, with what earlier emptyings left of them
        auto take = [&](int c, float (&v)[32]) {
          __syncwarp();
          tmem_load32(base + c, v);
          if (add) {
            float old[32];
            tmem_load32(sums + c, old);
            tmem_wait_load(v);
            tmem_wait_load(old);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += old[j];
          } else {
            tmem_wait_load(v);
          }
          if (!ok) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7fffffffu);
          }
        };
        auto put = [&](auto* q, size_t stride, int have) {      // to q, q + stride, ...; `have`: columns that exist
          using Q = std::remove_pointer_t<decltype(q)>;
          for (int c = 0; c < cols; c += 32) {
            float v[32];
            take(c, v);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < have) q[(c + j) * stride] = from_f32<Q>(v[j]);
          }
        };
        if (!last) {
          for (int c = 0; c < cols; c += 32) {
            float v[32];
            take(c, v);
            tmem_store32(sums + c, v);
          }
          tmem_wait_store();
        } else if (p.slot >= 0) {
          put(a.work + (size_t)p.slot * kSlotFloats + half * (kTileN * kTileK) + kl, kTileK, cols);
        } else if (sizeof(O) == 2 && a.ins % 8 == 0) {
          if constexpr (sizeof(O) == 2) {
            const int k8 = t.k0 + (warp - kEpilogueWarp0) * 32 + (lane & 24), n = t.n0 + (lane & 7);
            O* const q = static_cast<O*>(a.out) + (size_t)n * a.ins + k8;
            for (int c = 0; c < cols; c += 32) {
              float v[32];
              take(c, v);
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                const uint4 w = turn8<O>(v + j, lane);
                if (k8 < a.ins && n + c + j < a.outs) *reinterpret_cast<uint4*>(q + (size_t)(c + j) * a.ins) = w;
              }
            }
          }
        } else {
          put(static_cast<O*>(a.out) + (size_t)t.n0 * a.ins + k, a.ins, k < a.ins ? a.outs - t.n0 : 0);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(&sm.acc_empty[buf], 0);
      }
    }
  }

  // ---- the MMAs are done, in both CTAs: nobody's shared or tensor memory goes before ----
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (sm.failed) {   // arrivals that nobody waited for any more may still be on their way here
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 50000) {
    }
  }
  __syncwarp();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  cluster_sync();   // (the pair gives its tensor memory back together)
}

// Adds the runs of each tile that more than one pair worked on, in the order of their tokens.  A block takes 8 output
// features of one of the tile's two halves of input features, a thread four neighbouring input features.
template <class O>
__global__ void __launch_bounds__(256) wgrad_runs_kernel(const WgradArgs a) {
  __shared__ int s_p0, s_p1;
  const int r = blockIdx.y, half = blockIdx.z;
  const Tile t = tile_at(a, a.whole * a.pairs + r, half);
  if (threadIdx.x == 0) {
    // pairs [p0, p1]: the first whose run ends after the tile begins, the last whose run begins before the tile ends
    const long long total = (long long)a.rest * a.steps, first = (long long)r * a.steps, last = first + a.steps;
    int p0 = (int)(first * a.rest_pairs / total);
    while (p0 > 0 && p0 * total / a.rest_pairs > first) --p0;
    while ((p0 + 1) * total / a.rest_pairs <= first) ++p0;
    int p1 = p0;
    while (p1 + 1 < a.rest_pairs && (p1 + 1) * total / a.rest_pairs < last) ++p1;
    s_p0 = p0 * 2 + (r - (int)(p0 * total / a.rest_pairs / a.steps));   // its slot: the tile is the first or the second of its run
    s_p1 = p1 * 2;                                                      // the tile is the first of all later runs
  }
  __syncthreads();
  cudaGridDependencySynchronize();
  const int p0 = s_p0, p1 = s_p1;
  if (p1 <= p0) return;    // one pair did it all, straight to the output
  const int c = blockIdx.x * 8 + (threadIdx.x >> 5), kl = (threadIdx.x & 31) * 4, n = t.n0 + c, k = t.k0 + kl;
  if (c < t.boxes * 128 && n < a.outs && k < a.ins) {
    const float* const q = a.work + (half * kTileN + c) * kTileK + kl;
    float4 s = *reinterpret_cast<const float4*>(q + (size_t)p0 * kSlotFloats);
    for (int p = (p0 | 1) + 1; p <= p1; p += 8) {      // four loads under way at a time
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = p + 2 * i <= p1 ? *reinterpret_cast<const float4*>(q + (size_t)(p + 2 * i) * kSlotFloats) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) { s.x += v[i].x; s.y += v[i].y; s.z += v[i].z; s.w += v[i].w; }
    }
    O* const out = static_cast<O*>(a.out) + (size_t)n * a.ins + k;
    const float f[4] = {s.x, s.y, s.z, s.w};
    if (a.ins % 4 == 0) {     // (the output is a fresh allocation: its rows start where four elements do)
      struct alignas(4 * sizeof(O)) Four { O v[4]; };
      *reinterpret_cast<Four*>(out) = {{from_f32<O>(f[0]), from_f32<O>(f[1]), from_f32<O>(f[2]), from_f32<O>(f[3])}};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j < a.ins) out[j] = from_f32<O>(f[j]);
    }
  }
  const int col = t.share * a.bias_cols + threadIdx.x, nb = t.n0 + half * t.boxes * 64 + col;
  if (blockIdx.x == 0 && (int)threadIdx.x < a.bias_cols && col < t.boxes * 64 && nb < a.outs) {
    const float* const q = a.work + kPartFloats + half * kHalfN + col;
    float s = q[(size_t)p0 * kSlotFloats];
    for (int p = (p0 | 1) + 1; p <= p1; p += 2) s += q[(size_t)p * kSlotFloats];
    static_cast<O*>(a.bias)[nb] = from_f32<O>(s);
  }
}

// Rows of 16-bit elements copied to a pitch that TMA accepts (the source's is odd, or it starts off a 16-byte boundary).
__global__ void __launch_bounds__(256) repitch_kernel(const unsigned short* __restrict__ src, long long stride, uint4* __restrict__ dst,
                                                      long long rows, int cols, int chunks) {
  const long long n = rows * chunks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / chunks;
    const int col = (int)(i - row * chunks) * 8;
    const unsigned short* p = src + row * stride + col;
    unsigned h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = col + j < cols ? p[j] : 0u;
    dst[i] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {   // looked up at run time: the extension must load on machines without a driver
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess) p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

bool encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch_bytes,
            uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {inner, outer}, strides[1] = {pitch_bytes};
  const cuuint32_t box[2] = {box_inner, box_outer}, ones[2] = {1, 1};
  return encode_fn()(map, type, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a call is cut up.
struct Plan {
  int tiles_k, tiles, steps, pairs, whole, rest, rest_pairs, chunk;
  int longest;          // steps of the longest piece
  size_t work_bytes;
};
Plan make_plan(long long tokens, int outs, int ins, bool out_f32, int sms) {
  const bool scattered = !out_f32 && ins % 8 != 0;
  Plan p{};
  p.tiles_k = (ins + 2 * kTileK - 1) / (2 * kTileK);
  p.tiles = p.tiles_k * ((outs + kTileN - 1) / kTileN);
  p.steps = (int)((tokens + kStep - 1) / kStep);
  p.pairs = sms / 2;
  p.whole = p.tiles / p.pairs;
  p.rest = p.tiles % p.pairs;
  // The last wave's tiles are shared out where that saves more steps than the second kernel and the partial sums cost, at least
  // four steps for each pair: 24 steps, or any where the results' rows are off 16-byte boundaries, since whole tiles then go out
  // by single elements and shared ones through the second kernel in fours (fp16, us with 1 and with 24: 777 tokens 1000 x 1003 19.6
  // and 26.6; 1024 tokens 768 x 771 18.4 and 26.6; 2048 tokens 2000 x 2002 38.9 and 36.9; 4096 tokens 1000 x 1001 26.6 and 25.8).
  p.rest_pairs = p.rest;
  if (p.rest) {
    const long long total = (long long)p.rest * p.steps;
    long long n = total / 4 < p.pairs ? total / 4 : p.pairs;
    if (n > p.rest && p.steps - (total + n - 1) / n >= (scattered ? 1 : kMinSavedSteps)) p.rest_pairs = (int)n;
  }
  p.chunk = out_f32 ? kChunkStepsF32 : kChunkSteps16;
  p.longest = p.whole || p.rest_pairs == p.rest ? p.steps : (int)(((long long)p.rest * p.steps + p.rest_pairs - 1) / p.rest_pairs);
  p.work_bytes = p.rest_pairs > p.rest ? (size_t)p.rest_pairs * 2 * kSlotFloats * 4 : 0;
  return p;
}

template <class T, class O>
cudaError_t launch_typed(const CUtensorMap& dy, const CUtensorMap& codes, const WgradArgs& a, cudaStream_t stream) {
  const int smem = (int)sizeof(WgradSmem) + 1024;
  cudaError_t err = cudaFuncSetAttribute(wgrad_kernel<T, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (err != cudaSuccess) return err;
  wgrad_kernel<T, O><<<2 * (a.whole ? a.pairs : a.rest_pairs), kThreads, smem, stream>>>(dy, codes, a);
  err = cudaGetLastError();
  if (err != cudaSuccess || a.rest_pairs == a.rest) return err;
  // (its blocks may be set up while the first kernel still runs; they wait for its end before they read)
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kTileN / 8, a.rest, 2);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, wgrad_runs_kernel<O>, a);
}

}  // namespace

cudaError_t launch_act8_repitch(const void* src, long long stride, void* dst, long long rows, int cols, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  const int chunks = (cols + 7) / 8;
  const long long blocks = (rows * chunks + 255) / 256;
  repitch_kernel<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, stream>>>(static_cast<const unsigned short*>(src), stride,
                                                                                 static_cast<uint4*>(dst), rows, cols, chunks);
  return cudaGetLastError();
}

size_t act8_wgrad_work_bytes(long long tokens, int outs, int ins, int out_f32, int sms) {
  return tokens > 0 && outs > 0 && ins > 0 ? make_plan(tokens, outs, ins, out_f32 != 0, sms).work_bytes : 0;
}

// The copies run on the legacy stream, which torch's streams do not wait for: read and cleared only once the device is idle.
cudaError_t act8_wgrad_status(unsigned* words) {
  cudaError_t err = cudaDeviceSynchronize();
  if (err == cudaSuccess) err = cudaMemcpyFromSymbol(words, wgrad_status, sizeof(wgrad_status));
  if (err != cudaSuccess || words[0] == kOk) return err;
  const unsigned zeros[16] = {};
  err = cudaMemcpyToSymbol(wgrad_status, zeros, sizeof(zeros));
  return err != cudaSuccess ? err : cudaDeviceSynchronize();
}

cudaError_t act8_wgrad_status_block(void** block) { return cudaGetSymbolAddress(block, wgrad_status); }

cudaError_t launch_act8_wgrad(const void* grad, long long grad_stride, Held held, long long tokens, int outs, int ins, int dtype,
                              int out_f32, void* out, void* bias, void* work, int sms, cudaStream_t stream) {
  if (tokens <= 0 || outs <= 0 || ins <= 0 || tokens > (1ll << 31) - 64) return cudaErrorInvalidValue;
  if (dtype != kGradBF16 && dtype != kGradF16) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(grad) % 16 || grad_stride % 8 || reinterpret_cast<uintptr_t>(held.codes) % 16 || held.pitch % 32)
    return cudaErrorMisalignedAddress;
  if (!encode_fn()) return cudaErrorNotSupported;
  CUtensorMap map_dy, map_codes;
  const CUtensorMapDataType type = dtype == kGradBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (!encode(&map_dy, type, grad, outs, tokens, grad_stride * 2, 64, kStep, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode(&map_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, held.codes, held.pitch, tokens, held.pitch, kTileK, kStep, CU_TENSOR_MAP_SWIZZLE_NONE))
    return cudaErrorInvalidValue;
  const Plan plan = make_plan(tokens, outs, ins, out_f32, sms);
  if (plan.work_bytes && !work) return cudaErrorInvalidValue;
  int bias_cols = 0;
  if (bias) {
    bias_cols = 8;
    while (bias_cols * plan.tiles_k < kHalfN) bias_cols *= 2;
  }
  const WgradArgs a{held.scales, held.spitch, tokens, outs, ins, plan.tiles_k, plan.pairs, plan.whole, plan.rest, plan.rest_pairs,
                    plan.steps, plan.chunk, plan.chunk < plan.longest ? 1 : 0, 1u, bias_cols, out, bias, static_cast<float*>(work)};
  if (dtype == kGradBF16)
    return out_f32 ? launch_typed<__nv_bfloat16, float>(map_dy, map_codes, a, stream)
                   : launch_typed<__nv_bfloat16, __nv_bfloat16>(map_dy, map_codes, a, stream);
  return out_f32 ? launch_typed<__half, float>(map_dy, map_codes, a, stream)
                 : launch_typed<__half, __half>(map_dy, map_codes, a, stream);
}

}  // namespace grace
