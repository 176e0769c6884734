// Weight gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//   dW[n, k] = sum_m dY[m, n] x~[m, k]      db[n] = sum_m dY[m, n]
// without ever writing x~ to memory: its tiles are decoded on the way into the tensor core.
//
// The kernel computes dW^T tiles of 128 input features by 256 output features, D[k, n] += A[k, m] B[m, n], over steps of
// 64 tokens.  Both operands have the tokens as their contracted axis and lie in memory with the OTHER axis
// contiguous, which the tensor core takes as it is (MN-major operands, 128-byte rows of 64 elements in the 128-byte
// swizzle), so nothing is transposed:
//   B = dY     TMA boxes of 64 tokens x 64 output features land in the operand layout
//   A = x~     TMA brings the codes (64 tokens x 128 bytes); eight warps decode them and store the operand tile
// The checkpoint is the operand with the SHORT side (128 against 256) because its elements cost issue slots: 2.5
// instructions each, 64 * 128 * 2.5 / 128 lanes = 160 of the 512 cycles that the tensor core needs for the step.  For
// bf16 a code's sign bit and seven others are placed under a significand whose exponent already holds the scale, so
// decoding and scaling are one subtraction of two bf16 pairs; the result is exact.
//
// Roles: warp 0 loads (TMA; the four scale bytes a token by cp.async), warp 1 issues the MMAs, warps 2 - 3 add up the
// bias gradient (each CTA of a row of tiles takes its share of the 256 columns), warps 4 - 11 decode and, at the end,
// write the result from TMEM.  Few output tiles would leave SMs idle: then the tokens are split over a cluster of up
// to 8 CTAs, which add their partial tiles in rank order through distributed shared memory (no atomics: the same
// bits on every run).  Sums are fp32 throughout, rounded once to the output's type.
//
// Every wait is bounded; when one runs out the status block says which and the outputs are NaN.
#include <cooperative_groups.h>

#include "act8.cuh"
#include "act8.h"
#include "gradio.cuh"
#include "tensor_core.cuh"

namespace grace {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 384;
constexpr int kTileK = 128;            // input features of a tile: MMA M
constexpr int kTileN = 256;            // output features of a tile: MMA N
constexpr int kStep = 64;              // tokens of a step
constexpr int kBoxBytes = kStep * 128; // 64 tokens x 64 features of 16 bits
constexpr int kBBytes = 4 * kBoxBytes;
constexpr int kCodeBytes = kStep * kTileK;
constexpr int kABytes = 2 * kBoxBytes;
constexpr int kStages = 4, kAStages = 3;
constexpr int kDecodeWarp0 = 4, kDecodeWarps = 8;
constexpr unsigned long long kTimeoutNs = 2000000000ull;
constexpr unsigned kTmemCols = 256;

struct __align__(1024) WgradSmem {
  unsigned char b[kStages][kBBytes];        // reused at the end: [256][128] fp32 partial tile for the cluster's other CTAs
  unsigned char a[kAStages][kABytes];
  unsigned char codes[kStages][kCodeBytes];
  unsigned scales[kStages][kStep];          // four scale bytes of a token: the tile's 128 features
  float bias[kTileN];
  unsigned long long full[kStages], empty[kStages], a_full[kAStages], a_empty[kAStages], done;
  unsigned tmem_base;
  unsigned ok;
};
static_assert(kStages * kBBytes >= kTileN * kTileK * 4, "the partial tile reuses the operand ring");

struct WgradArgs {
  const unsigned char* scales;
  int spitch;
  long long tokens;
  int outs, ins;        // N, K
  int steps;            // of 64 tokens, over all tokens
  int bias_cols;        // columns of the 256 that a CTA adds up (a power of two), 0: no bias gradient
  void* out;
  void* bias;
};

// The status block of the bounded waits (common.cuh), one for each device, sticky until act8_wgrad_status clears it.  A
// symbol and not an allocation, so that the first call may be made while a graph is being captured.
__device__ unsigned wgrad_status[16];

__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"((unsigned)accum) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(void* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Eight codes as a 16-byte operand chunk.
__device__ __forceinline__ uint4 decode8(uint2 c, unsigned s, __nv_bfloat16) {
  // exponent field s + 7: 2^(s - 127) * 128 * (1 + m / 128) = (128 + m) steps
  const unsigned base = s == 255u ? 0x7fc07fc0u : ((s + 7u) << 7) * 0x10001u;
  unsigned r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned v = __byte_perm(j < 2 ? c.x : c.y, 0u, (j & 1) ? 0x4342 : 0x4140);   // two codes, 16 bits each
    const unsigned hi = (v & 0x007f007fu) | base;          // (128 + low seven bits) steps
    const unsigned lo = (v & 0x00800080u) + base;          // 128 steps, or 256 for a negative code
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&hi), *reinterpret_cast<const __nv_bfloat162*>(&lo));
    r[j] = *reinterpret_cast<const unsigned*>(&d);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint4 decode8(uint2 c, unsigned s, __half) {   // (fp16's exponent range is too short for that)
  float v[8];
  act8_decode(c, s, v);
  Chunk8<__half> h;
  h.set(v);
  return h.w;
}

template <class T> constexpr uint32_t instruction_desc() {
  constexpr uint32_t f = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(kTileK >> 4) << 24);   // N is added at run time
}

template <class T, class O>
__global__ void __launch_bounds__(kThreads, 1) wgrad_kernel(const __grid_constant__ CUtensorMap map_dy,
                                                            const __grid_constant__ CUtensorMap map_codes, const WgradArgs a) {
  extern __shared__ unsigned char raw[];
  WgradSmem& sm = *reinterpret_cast<WgradSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Status status{wgrad_status};
  const int splits = gridDim.z, split = blockIdx.z;      // the cluster: (1, 1, splits)
  const int k0 = blockIdx.x * kTileK, n0 = blockIdx.y * kTileN;
  const int step0 = (int)((long long)a.steps * split / splits);
  const int nsteps = (int)((long long)a.steps * (split + 1) / splits) - step0;
  const int boxes = min(4, (a.outs - n0 + 63) / 64);     // 64-feature blocks of this tile that exist
  const bool has_bias = a.bias_cols != 0;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1 + 32);
      mbar_init(&sm.empty[s], 1 + kDecodeWarps + (has_bias ? 2 : 0));
    }
    for (int s = 0; s < kAStages; ++s) { mbar_init(&sm.a_full[s], kDecodeWarps); mbar_init(&sm.a_empty[s], 1); }
    mbar_init(&sm.done, 1);
    sm.ok = 1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ---- loads ----
    bool ok = true;
    int st = 0;
    for (; st < nsteps; ++st) {
      const int slot = st % kStages;
      if (st >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[slot], (st / kStages - 1) & 1, kTimeoutNs, status, 100 + slot));
      if (!ok) break;
      const int m = (step0 + st) * kStep;
      if (lane == 0) {
        mbar_expect_tx(&sm.full[slot], boxes * kBoxBytes + kCodeBytes);
        for (int j = 0; j < boxes; ++j) tma_load_2d(&sm.b[slot][j * kBoxBytes], &map_dy, n0 + j * 64, m, &sm.full[slot]);
        tma_load_2d(&sm.codes[slot][0], &map_codes, k0, m, &sm.full[slot]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const long long row = m + lane + 32 * i;
        const bool in = row < a.tokens;
        cp_async4(&sm.scales[slot][lane + 32 * i], a.scales + (in ? row : 0) * a.spitch + (k0 >> 5), in);   // past the end: zeros
      }
      cp_async_arrive(&sm.full[slot]);
    }
    if (!ok)   // a consumer gave up: the loads that were issued must land before the shared memory is let go
      for (int s = st > kStages ? st - kStages : 0; s < st; ++s) mbar_wait(&sm.full[s % kStages], (s / kStages) & 1, kTimeoutNs, status, 400);
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 1) {
    // ---- MMAs ----
    if (lane == 0) {
      const uint32_t idesc = instruction_desc<T>() | ((uint32_t)(boxes * 8) << 17);
      for (int st = 0; st < nsteps; ++st) {
        const int slot = st % kStages, as = st % kAStages;
        if (!mbar_wait(&sm.full[slot], (st / kStages) & 1, kTimeoutNs, status, 200 + slot) ||
            !mbar_wait(&sm.a_full[as], (st / kAStages) & 1, kTimeoutNs, status, 300 + as)) {
          sm.ok = 0;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(sm.a[as]), b_addr = smem_u32(sm.b[slot]);
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk)   // 16 tokens: two groups of eight 128-byte rows; the next 64 features one box further
          umma_f16(tmem, smem_desc(a_addr + kk * 2048, kBoxBytes, 1024, 2), smem_desc(b_addr + kk * 2048, kBoxBytes, 1024, 2), idesc,
                   st > 0 || kk > 0);
        umma_commit(&sm.a_empty[as]);
        umma_commit(&sm.empty[slot]);
      }
      umma_commit(&sm.done);
    }
  } else if (warp < kDecodeWarp0) {
    // ---- bias gradient: this CTA's share of the tile's columns, two a thread, rows dealt to `groups` threads ----
    if (has_bias) {
      const int t = tid - 64, pairs = a.bias_cols >> 1;
      const int groups = min(32, 64 / min(64, pairs)), own = t / groups, sub = t % groups;
      const int c0 = blockIdx.x * a.bias_cols;             // first column; CTAs past the 256th column have none
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      bool ok = true;
      for (int st = 0; st < nsteps; ++st) {
        const int slot = st % kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.full[slot], (st / kStages) & 1, kTimeoutNs, status, 500 + slot));
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pair = own + 64 * h, col = c0 + pair * 2;
          if (pair < pairs && col < boxes * 64) {
            const unsigned char* p = &sm.b[slot][(col >> 6) * kBoxBytes + (col & 7) * 2];
            for (int m = sub; m < kStep; m += groups) {
              const unsigned v = *reinterpret_cast<const unsigned*>(p + m * 128 + ((((col >> 3) & 7) ^ (m & 7)) << 4));
              const unsigned short lo = (unsigned short)v, hi = (unsigned short)(v >> 16);
              acc[2 * h] += to_f32<T>(*reinterpret_cast<const T*>(&lo));
              acc[2 * h + 1] += to_f32<T>(*reinterpret_cast<const T*>(&hi));
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[slot]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int o = groups >> 1; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      if (sub == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pair = own + 64 * h, col = c0 + pair * 2;
          if (pair < pairs && col < kTileN) {
            sm.bias[col] = acc[2 * h];
            sm.bias[col + 1] = acc[2 * h + 1];
          }
        }
      }
    }
  } else {
    // ---- decode: a thread takes eight codes (a 16-byte operand chunk) of four tokens a step ----
    const int t = tid - kDecodeWarp0 * 32, chunk = t & 15, row0 = t >> 4;
    for (int st = 0; st < nsteps; ++st) {
      const int slot = st % kStages, as = st % kAStages;
      bool ok = mbar_wait(&sm.full[slot], (st / kStages) & 1, kTimeoutNs, status, 600 + slot);
      if (ok && st >= kAStages) ok = mbar_wait(&sm.a_empty[as], (st / kAStages - 1) & 1, kTimeoutNs, status, 700 + as);
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = row0 + 16 * i;
        const uint2 c = *reinterpret_cast<const uint2*>(&sm.codes[slot][m * kTileK + chunk * 8]);
        const unsigned s = (sm.scales[slot][m] >> ((chunk >> 2) * 8)) & 0xffu;
        *reinterpret_cast<uint4*>(&sm.a[as][(chunk >> 3) * kBoxBytes + m * 128 + (((chunk & 7) ^ (m & 7)) << 4)]) = decode8(c, s, T{});
      }
      fence_async_all();   // the tensor core reads the tile through the async proxy
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.empty[slot]);
        mbar_arrive(&sm.a_full[as]);
      }
    }
  }

  // ---- result: TMEM lane = input feature, column = output feature ----
  __syncwarp();
  const bool done = mbar_wait(&sm.done, 0, 2 * kTimeoutNs, status, 800);   // (also: no MMA reads the rings any more)
  if (!done) sm.ok = 0;
  __syncthreads();
  tc_fence_after();
  bool good = sm.ok && !status.failed();
  const float nan = __uint_as_float(0x7fffffffu);
  O* const out = static_cast<O*>(a.out);
  if (warp >= kDecodeWarp0) {
    const int quarter = warp & 3, half = (warp - kDecodeWarp0) >> 2;      // a warp reads its own quarter of the TMEM lanes
    const int kl = quarter * 32 + lane, k = k0 + kl;
    float* const part = reinterpret_cast<float*>(sm.b[0]);
    for (int c = half * 128; c < half * 128 + 128 && c < boxes * 64; c += 32) {
      uint32_t v[32];
      asm volatile(
          "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
          "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
          : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
            "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
            "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
            "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
          : "r"(tmem + c + ((uint32_t)(quarter * 32) << 16)));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (splits == 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (k < a.ins && n0 + c + j < a.outs)
            out[(size_t)(n0 + c + j) * a.ins + k] = from_f32<O>(good ? __uint_as_float(v[j]) : nan);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) part[(c + j) * kTileK + kl] = __uint_as_float(v[j]);
      }
    }
  }
  if (splits == 1) {
    if (has_bias) {
      const int c = blockIdx.x * a.bias_cols + tid;
      if (tid < a.bias_cols && c < kTileN && n0 + c < a.outs) static_cast<O*>(a.bias)[n0 + c] = from_f32<O>(good ? sm.bias[c] : nan);
    }
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int r = 0; r < splits; ++r) good = good && *cluster.map_shared_rank(&sm.ok, r) != 0;
    const int per = (kTileN + splits - 1) / splits, c_end = min(min((split + 1) * per, kTileN), boxes * 64);
    for (int i = tid; i < per * (kTileK / 4); i += kThreads) {     // four input features of one column
      const int c = split * per + i / (kTileK / 4), kl = (i % (kTileK / 4)) * 4;
      const int n = n0 + c, k = k0 + kl;
      if (c >= c_end || n >= a.outs || k >= a.ins) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < splits; ++r) {
        const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(reinterpret_cast<float*>(sm.b[0]) + c * kTileK + kl, r));
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
      const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j < a.ins) out[(size_t)n * a.ins + k + j] = from_f32<O>(good ? s[j] : nan);
    }
    if (has_bias && split == 0) {
      const int c = blockIdx.x * a.bias_cols + tid;
      if (tid < a.bias_cols && c < kTileN && n0 + c < a.outs) {
        float s = 0.f;
        for (int r = 0; r < splits; ++r) s += *cluster.map_shared_rank(&sm.bias[c], r);
        static_cast<O*>(a.bias)[n0 + c] = from_f32<O>(good ? s : nan);
      }
    }
    cluster.sync();   // nobody's shared memory goes before its readers are done
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
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

template <class T, class O>
cudaError_t launch_typed(const CUtensorMap& dy, const CUtensorMap& codes, const WgradArgs& a, dim3 grid, cudaStream_t stream) {
  const int smem = (int)sizeof(WgradSmem) + 1024;
  cudaError_t err = cudaFuncSetAttribute(wgrad_kernel<T, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = grid.z;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, wgrad_kernel<T, O>, dy, codes, a);
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

cudaError_t act8_wgrad_status(unsigned* words) {
  cudaError_t err = cudaMemcpyFromSymbol(words, wgrad_status, sizeof(wgrad_status));   // waits for the device's work
  if (err != cudaSuccess || words[0] == kOk) return err;
  const unsigned zeros[16] = {};
  return cudaMemcpyToSymbol(wgrad_status, zeros, sizeof(zeros));
}

cudaError_t launch_act8_wgrad(const void* grad, long long grad_stride, Held held, long long tokens, int outs, int ins, int dtype,
                              int out_f32, void* out, void* bias, int sms, cudaStream_t stream) {
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
  const int kt = (ins + kTileK - 1) / kTileK, nt = (outs + kTileN - 1) / kTileN;
  const int steps = (int)((tokens + kStep - 1) / kStep);
  int splits = 1;
  while (splits < 8 && (long long)kt * nt * (splits + 1) <= sms && steps / (splits + 1) >= 4) ++splits;
  int bias_cols = 0;
  if (bias) {
    bias_cols = 2;
    while (bias_cols * kt < kTileN) bias_cols *= 2;
  }
  const WgradArgs a{held.scales, held.spitch, tokens, outs, ins, steps, bias_cols, out, bias};
  const dim3 grid(kt, nt, splits);
  if (dtype == kGradBF16)
    return out_f32 ? launch_typed<__nv_bfloat16, float>(map_dy, map_codes, a, grid, stream)
                   : launch_typed<__nv_bfloat16, __nv_bfloat16>(map_dy, map_codes, a, grid, stream);
  return out_f32 ? launch_typed<__half, float>(map_dy, map_codes, a, grid, stream)
                 : launch_typed<__half, __half>(map_dy, map_codes, a, grid, stream);
}

}  // namespace grace
