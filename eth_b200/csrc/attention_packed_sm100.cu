// Flash attention over packed documents for sm_100a: forward and backward on tcgen05 tensor cores with
// TMEM accumulators, documents of any length one behind the other on one row axis, grouped heads.
//
// A host-built work list names (document start, length, tile) per unit of work, heaviest first; tiles
// are aligned to their document, so no tile mixes documents and nothing of one document reaches
// another. Where a tile runs over its document's end, its rows behind the end are cleared in shared
// memory before they become summands of an MMA.
//
// Forward. One CTA owns two 128-row query tiles and streams the key/value tiles once for both:
//   warp 0      TMA producer: Q (once), then K_j / V_j tiles into a ring of shared-memory stages.
//   warp 1      MMA issuer:   S_t = Q_t K_j^T  (operands in shared memory, accumulator in TMEM),
//               O_t += P_t V_j (P_t read from TMEM, V_j from shared memory as an MN-major operand).
//   warps 2-5   softmax of query tile 0, warps 6-9 softmax of query tile 1: one thread per query
//               row; online softmax in the exp2 domain, P written back to TMEM as packed 16-bit
//               (aliasing the scores), the O accumulator rescaled only when the running maximum grew
//               by more than 2^8 (exact after the final normalisation).
// The two tiles are the same rows of two heads of a group where the group is even (both then meet the
// same number of key tiles under the causal mask, and a document of up to 128 rows fills both), else
// two consecutive tiles of one head.
//
// TMEM map (512 columns): S_0/P_0 [0,128)  S_1/P_1 [128,256)  O_0 [256,256+D)  O_1 [384,384+D).
//
// P and dS are rounded to the input type, as the tensor core takes both operands in one type; the
// sums, the softmax statistics and all accumulators are fp32.
#include "attention_packed_sm100.cuh"
#include "gemm_sm100.cuh"
#include "sm100_common.cuh"

#include <atomic>
#include <mutex>

namespace ethb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 128;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) ==
            cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(sym);
  });
  return fn;
}

// 3-D map over a [rows, heads, head_dim] view: dims {d, rows, heads}, box {64, 128, 1}. A tile may start
// at any row; rows beyond the last read as 0.
cudaError_t make_tmap_rhd(CUtensorMap* map, const void* base, int dtype, int d, int rows, int heads,
                          const int64_t strides[2]) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  ensure_thread_context();
  ETHB_RETURN_IF((reinterpret_cast<uintptr_t>(base) & 15) != 0 || strides[0] % 8 != 0 || strides[1] % 8 != 0,
                 cudaErrorMisalignedAddress, "packed attention: base and strides must be multiples of 16 bytes");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(heads)};
  const cuuint64_t gstr[2] = {static_cast<cuuint64_t>(strides[0]) * 2, static_cast<cuuint64_t>(strides[1]) * 2};
  const cuuint32_t box[3] = {64, kTile, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        3, const_cast<void*>(base), dims, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  ETHB_RETURN_IF(r != CUDA_SUCCESS, cudaErrorInvalidValue, "cuTensorMapEncodeTiled (packed attention)");
  return cudaSuccess;
}

// Where a wait that gave up leaves its mark: the device's status word, which the host reads, and a flag of
// the CTA, by which its roles stop. They do not stop for the status word itself, as a mark that an earlier
// kernel has left there would leave results of this one unwritten.
struct Marks {
  int* status;
  int* gave_up;
};
__device__ __forceinline__ void give_up(int* flag) { *reinterpret_cast<volatile int*>(flag) = 1; }
__device__ __forceinline__ bool marked_wait(uint64_t* bar, uint32_t parity, const Marks& marks, int code) {
  const bool got = mbar_wait(bar, parity, marks.status, code);
  if (!got) give_up(marks.gave_up);
  return got;
}
// A wait whose outcome all lanes of the warp share, so that a timeout cannot split a warp (or, through
// wg_and, a warpgroup) between leaving and going on to the next warp-wide or group-wide operation.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Marks& marks, int code) {
  return __all_sync(0xffffffffu, marked_wait(bar, parity, marks, code));
}
// For the forward kernel, whose roles set the flag behind their loops: with it in every wait the softmax loop
// is compiled otherwise (one document of 8192, 32 / 8 heads of 128: 497 us against 485).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
}

__device__ __forceinline__ uint32_t pack_pair(float a, float b, int dtype) {
  return pack2(a, b, dtype);
}

// 2^x on the FMA pipe: x = i + f with i the nearest whole number, 2^f on [-1/2, 1/2] by a polynomial
// (minimax in relative error, found by Remez exchange), 2^i built in the exponent field. The softmax
// warps take part of their exponentials this way: 16 special-function results per clock and SM are the
// longest step of a score tile, the FMA pipe is idle then. Degree 4 is off by 2.7e-6 at most. Below
// x = -126.5 the result is 0 (the exponent field of i = -127 is that of 0); NaN stays NaN.
__device__ __forceinline__ Pair exp2_poly(Pair x) {
  float a, b;
  split(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  x = pair(a, b);
  const float magic = 12582912.f;   // 1.5 * 2^23: the sum's low mantissa bits hold the rounded x
  const Pair r = x + pair(magic, magic);
  const Pair f = x + (pair(magic, magic) + r * pair(-1.f, -1.f));
  Pair y = pair(0.0095701f, 0.0095701f);
  y = fma2(y, f, pair(0.05591786f, 0.05591786f));
  y = fma2(y, f, pair(0.24024745f, 0.24024745f));
  y = fma2(y, f, pair(0.69312181f, 0.69312181f));
  y = fma2(y, f, pair(0.99999926f, 0.99999926f));
  split(r, a, b);
  return y * pair(__int_as_float((__float_as_int(a) << 23) + 0x3f800000),
                  __int_as_float((__float_as_int(b) << 23) + 0x3f800000));
}
__device__ __forceinline__ Pair exp2_sfu(Pair x) {
  float a, b;
  split(x, a, b);
  return pair(exp2f(a), exp2f(b));
}
// Pair `i` of a row of scores: kPolyPairs out of four take the FMA pipe.
template <int kPolyPairs>
__device__ __forceinline__ Pair exp2_mixed(int i, Pair x) {
  return (i & 3) < kPolyPairs ? exp2_poly(x) : exp2_sfu(x);
}
__device__ __forceinline__ uint32_t pack_pair(Pair p, int dtype) {
  float a, b;
  split(p, a, b);
  return pack2(a, b, dtype);
}
// Measured: dK / dV and dQ of 8192 rows in five documents, 32 / 8 heads of 128: 295 and 226 us with none, 290 and
// 227 with a quarter, 289 and 236 with a half, 313 and 245 with three quarters; nine documents, 16 heads of 128: 112
// and 80, 109 and 80, 110 and 83, 116 and 85. (In the forward, whose registers are full, a quarter took 93 us in
// place of 74 at nine documents.)
constexpr int kBwdPoly = 1;

// Clears rows [first, 128) of a tile that a TMA load has written (kHalves blocks of 128 rows x 128
// bytes; the swizzle permutes inside a row only) and makes that visible to the tensor core's reads.
// Executed by one warp; the caller signals the tile afterwards.
template <int kHalves>
__device__ __forceinline__ void clear_tail(uint8_t* tile, int first, int lane) {
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
    for (int c = first * 8 + lane; c < kTile * 8; c += 32)
      reinterpret_cast<uint4*>(tile + h * 16384)[c] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
}

// Clears rows [first, rows) of a [rows, heads, D] 16-bit output: part `part` of `parts`, thread `tid` of `threads`.
template <int D>
__device__ __forceinline__ void clear_rows(void* base, int64_t row_stride, int64_t head_stride, int first, int rows, int heads,
                                           int part, int parts, int tid, int threads) {
  constexpr int kChunks = D / 8;
  const int64_t total = static_cast<int64_t>(rows - first) * heads * kChunks;
  for (int64_t i = static_cast<int64_t>(part) * threads + tid; i < total; i += static_cast<int64_t>(parts) * threads) {
    const int c = static_cast<int>(i % kChunks);
    const int64_t rh = i / kChunks;
    uint16_t* at = reinterpret_cast<uint16_t*>(base) + (first + rh / heads) * row_stride + (rh % heads) * head_stride;
    reinterpret_cast<uint4*>(at)[c] = make_uint4(0, 0, 0, 0);
  }
}

// Four lanes hold four 16-byte chunks of a row each; afterwards lane l of them holds chunk l of the
// four rows.
__device__ __forceinline__ void transpose4(uint4 (&c)[4], int lane) {
  const auto swap = [&](uint4& lo, uint4& hi, int bit) {   // the off-diagonal chunk of a 2 x 2 block
    const bool up = lane & bit;
    uint4 x = up ? lo : hi;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, bit);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, bit);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, bit);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, bit);
    if (up) lo = x; else hi = x;
  };
  swap(c[0], c[1], 1);
  swap(c[2], c[3], 1);
  swap(c[0], c[2], 2);
  swap(c[1], c[3], 2);
}

// Columns [col, col + 32) of this warp's 32 accumulator rows to a 16-bit output whose row r begins at
// rows + r * stride; row r is written where r < valid. A thread reads one row from TMEM; stored like
// that, every 16-byte store of a warp would touch 32 lines (4000 cycles for a 128 x 128 pair of
// accumulators). Four lanes exchange their chunks first and write 64 bytes of a row together.
template <int DT>
__device__ __forceinline__ void store_columns(uint32_t acc, int col, uint16_t* rows, int64_t stride, int first, int valid,
                                              float mul, int lane) {
  uint32_t r[32];
  __syncwarp();
  tmem_ld_32x32b_x32(acc + col, r);
  tmem_ld_wait();
  uint4 c[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    c[q].x = pack_pair(__uint_as_float(r[q * 8 + 0]) * mul, __uint_as_float(r[q * 8 + 1]) * mul, DT);
    c[q].y = pack_pair(__uint_as_float(r[q * 8 + 2]) * mul, __uint_as_float(r[q * 8 + 3]) * mul, DT);
    c[q].z = pack_pair(__uint_as_float(r[q * 8 + 4]) * mul, __uint_as_float(r[q * 8 + 5]) * mul, DT);
    c[q].w = pack_pair(__uint_as_float(r[q * 8 + 6]) * mul, __uint_as_float(r[q * 8 + 7]) * mul, DT);
  }
  transpose4(c, lane);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = first + (lane & ~3) + k;
    if (row < valid) reinterpret_cast<uint4*>(rows + row * stride + col)[lane & 3] = c[k];
  }
}
// All D columns, and what their rounding took off to a second output that is laid out alike. A call of its
// own: inlined, it costs the forward's softmax loop registers that it does not have.
template <int D, int DT>
__device__ __noinline__ void store_with_residue(uint32_t acc, uint16_t* rows, int64_t stride, uint16_t* left,
                                                int64_t left_stride, int first, int valid, float mul, int lane) {
#pragma unroll 1
  for (int col = 0; col < D; col += 32) {
    uint32_t r[32];
    __syncwarp();
    tmem_ld_32x32b_x32(acc + col, r);
    tmem_ld_wait();
    uint4 c[4], d[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __uint_as_float(r[q * 8 + 2 * e]) * mul, y = __uint_as_float(r[q * 8 + 2 * e + 1]) * mul;
        hi[e] = pack_pair(x, y, DT);
        const float2 h = unpack2(hi[e], DT);
        lo[e] = pack_pair(x - h.x, y - h.y, DT);
      }
      c[q] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      d[q] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    transpose4(c, lane);
    transpose4(d, lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = first + (lane & ~3) + k;
      if (row >= valid) continue;
      reinterpret_cast<uint4*>(rows + row * stride + col)[lane & 3] = c[k];
      reinterpret_cast<uint4*>(left + row * left_stride + col)[lane & 3] = d[k];
    }
  }
}
// The same in fp32 (128 bytes of a row, two halves of 16 columns).
__device__ __forceinline__ void store_columns_f32(uint32_t acc, int col, float* rows, int64_t stride, int first, int valid,
                                                  float mul, int lane) {
  uint32_t r[32];
  __syncwarp();
  tmem_ld_32x32b_x32(acc + col, r);
  tmem_ld_wait();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 c[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = half * 16 + q * 4;
      c[q] = make_uint4(__float_as_uint(__uint_as_float(r[e]) * mul), __float_as_uint(__uint_as_float(r[e + 1]) * mul),
                        __float_as_uint(__uint_as_float(r[e + 2]) * mul), __float_as_uint(__uint_as_float(r[e + 3]) * mul));
    }
    transpose4(c, lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = first + (lane & ~3) + k;
      if (row < valid) reinterpret_cast<uint4*>(rows + row * stride + col + half * 16)[lane & 3] = c[k];
    }
  }
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

// The dynamic shared memory limit is a property of a kernel on a device; setting it again is harmless.
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// ==============================================================================================
// forward
// ==============================================================================================
template <int D> struct FwdCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kQBytes = 2 * kHalves * 16384;       // two query tiles
  // K and V tiles travel through one ring of equal slots in the order K_0 V_0 K_1 V_1 ...: a K
  // slot is free again as soon as both score MMAs of its tile are done, a whole iteration before
  // the V slot of the same tile, so five slots keep the loads a full iteration ahead of their use.
  static constexpr int kSlotBytes = kHalves * 16384;
  static constexpr int kSlots = (D == 128) ? 5 : 8;
  static constexpr int kSmemBytes = kQBytes + kSlots * kSlotBytes + 1024 + 512;
  static constexpr int kThreads = 320;
};

struct FwdBarriers {
  uint4 answer[2];        // of the launch control, see NextBlock
  uint64_t answer_full[2];
  uint64_t answer_read[2];
  uint64_t q_full;
  uint64_t q_free;        // the unit's last score MMAs have read Q
  uint64_t tail_full;     // the last V tile of a document has landed, rows behind its end not yet cleared
  uint64_t kv_full[8];
  uint64_t kv_empty[8];
  uint64_t s_full[2];
  uint64_t p_half[8];     // [tile * 4 + quarter]: 32 more P columns of a tile are written
  uint64_t o_done[2];
  uint32_t tmem_base;
  int gave_up;            // see Marks
};

// A CTA that is done with its block of the grid takes over blocks that have not been launched yet (cluster
// launch control): the hardware's dispatch in index order, heaviest first, stays as it is, and the set-up
// of TMEM, barriers and descriptors is paid once per SM. One thread asks for the next block while the
// current one is worked on; the answer lands in shared memory like a TMA load.
__device__ __forceinline__ void ask_next_block(FwdBarriers* bars, int it) {
  mbar_expect_tx(&bars->answer_full[it & 1], 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(&bars->answer[it & 1])), "r"(smem_u32(&bars->answer_full[it & 1]))
               : "memory");
}
// All lanes of a warp: the block that follows the `it`-th of this CTA, -1 if there is none.
__device__ __forceinline__ int next_block(FwdBarriers* bars, int it, int lane, int* status) {
  if (!warp_wait(&bars->answer_full[it & 1], static_cast<uint32_t>(it >> 1) & 1, status, kStatusTimeoutFull)) return -1;
  uint32_t taken = 0, x = 0;
  asm volatile(
      "{\n"
      ".reg .b128 r;\n"
      ".reg .pred p;\n"
      "ld.shared.b128 r, [%2];\n"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n"
      "}\n"
      : "=r"(taken), "+r"(x)
      : "r"(smem_u32(&bars->answer[it & 1]))
      : "memory");
  fence_proxy_async();   // the answer has been read before the next one may be written over it
  __syncwarp();
  if (lane == 0) mbar_arrive(&bars->answer_read[it & 1]);
  return taken != 0 ? static_cast<int>(x) : -1;
}

template <int kSlots> struct FwdRing {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == kSlots) { slot = 0; phase ^= 1; }
  }
};

// What a block of the grid stands for.
template <bool kPair> struct FwdUnit {
  PackedTile w;
  int head0, kv_head, kv_tiles;
  int qt0, qt1, n0, n1;      // query tiles inside the document and the key tiles they meet
  int n, tail_rows;
  __device__ __forceinline__ FwdUnit(const PackedAttnArgs& p, int block) {
    const int units = kPair ? p.heads / 2 : p.heads;
    w = p.tiles[block / units];
    const int unit = block % units;
    head0 = kPair ? 2 * unit : unit;                 // head of tile t: head0 + t when heads are paired
    kv_head = head0 / (p.heads / p.kv_heads);
    kv_tiles = (w.len + kTile - 1) / kTile;
    qt0 = kPair ? w.tile : 2 * w.tile;
    qt1 = kPair ? w.tile : 2 * w.tile + 1;
    n0 = p.causal ? qt0 + 1 : kv_tiles;
    n1 = qt1 >= kv_tiles ? 0 : p.causal ? qt1 + 1 : kv_tiles;
    n = max(n0, n1);
    // rows of the last key tile that belong to the document, if that tile is met: V rows behind them are
    // cleared, since a probability of 0 times whatever stands there would still be NaN for an infinity
    tail_rows = n == kv_tiles ? w.len - (kv_tiles - 1) * kTile : kTile;
  }
};

template <int D, int DT, bool kPair>
__global__ void __launch_bounds__(320, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, const PackedAttnArgs p) {
  using C = FwdCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + C::kQBytes;
  FwdBarriers* bars = reinterpret_cast<FwdBarriers*>(sKV + C::kSlots * C::kSlotBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // blocks of the grid: [work units, heaviest first][rows behind the last document to clear]
  const int work = p.num_tiles * (kPair ? p.heads / 2 : p.heads);

  if (threadIdx.x == 0) {
    bars->gave_up = 0;
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->answer_full[b], 1);
      mbar_init(&bars->answer_read[b], 10);   // every warp
    }
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_free, 1);
    mbar_init(&bars->tail_full, 1);
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&bars->kv_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->s_full[t], 1);
      for (int q = 0; q < 4; ++q) mbar_init(&bars->p_half[4 * t + q], 4);   // one arrival per softmax warp
      mbar_init(&bars->o_done[t], 1);
    }
    fence_mbar_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 1) tmem_alloc(&bars->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  // Every role walks over the CTA's blocks on its own; barrier parities run on what it has counted so far.
  const auto each_block = [&](auto one) {
    for (int it = 0, block = blockIdx.x; block >= 0; ++it) {
      one(it, block);
      block = next_block(bars, it, lane, p.status);
      if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&bars->gave_up) != 0)) break;
    }
  };
  if (warp == 0) {
    FwdRing<C::kSlots> ring;
    uint32_t units = 0, cuts = 0;
    each_block([&](int it, int block) {
      // Asked for when this block's last loads are on their way: early enough for the answer to be there
      // when the others need it, late enough that a CTA with a long block does not take another one
      // that a CTA about to finish could start on.
      const auto ask = [&] {
        if (warp_wait(&bars->answer_read[it & 1], (static_cast<uint32_t>(it >> 1) & 1) ^ 1, p.status,
                      kStatusTimeoutEmpty) && elect_one())
          ask_next_block(bars, it);
        __syncwarp();
      };
      if (block >= work) return ask();
      const FwdUnit<kPair> u(p, block);
      const PackedTile& w = u.w;
      const int n = u.n;
      // ---------------------------------------------------------------- producer
      const bool cut = u.tail_rows < kTile;
      bool ok = warp_wait(&bars->q_free, (units & 1) ^ 1, p.status, kStatusTimeoutEmpty);
      if (ok && elect_one()) {
        mbar_expect_tx(&bars->q_full, C::kQBytes);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
            tma_load_3d(sQ + (t * C::kHalves + h) * 16384, &tq, &bars->q_full, h * 64,
                        w.start + (t == 0 ? u.qt0 : u.qt1) * kTile, kPair ? u.head0 + t : u.head0);
      }
      __syncwarp();
      int last_slot = 0;
      for (int i = 0; i < 2 * n && ok; ++i) {   // item 2j is K_j, item 2j + 1 is V_j
        ok = warp_wait(&bars->kv_empty[ring.slot], ring.phase ^ 1, p.status, kStatusTimeoutEmpty);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = sKV + ring.slot * C::kSlotBytes;
          uint64_t* full = cut && i == 2 * n - 1 ? &bars->tail_full : &bars->kv_full[ring.slot];
          mbar_expect_tx(full, C::kSlotBytes);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
            tma_load_3d(dst + h * 16384, (i & 1) ? &tv : &tk, full, h * 64, w.start + (i >> 1) * kTile, u.kv_head);
        }
        __syncwarp();
        last_slot = ring.slot;
        ring.advance();
      }
      ask();
      if (cut && ok) {
        ok = warp_wait(&bars->tail_full, cuts & 1, p.status, kStatusTimeoutFull);
        ++cuts;
        if (ok) {
          clear_tail<C::kHalves>(sKV + last_slot * C::kSlotBytes, u.tail_rows, lane);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->kv_full[last_slot]);
        }
      }
      if (!ok) give_up(&bars->gave_up);
      ++units;
    });
  } else if (warp == 1) {
    FwdRing<C::kSlots> ring;
    uint32_t units = 0;
    int base0 = 0, base1 = 0;            // key tiles that the two query tiles have met
    each_block([&](int, int block) {
      if (block >= work) return;
      const FwdUnit<kPair> u(p, block);
      const PackedTile& w = u.w;
      const int n = u.n;
      // ---------------------------------------------------------------- MMA issuer
      if (elect_one()) {
        const int fmt = DT == kBF16 ? 1 : 0;
        const uint32_t idesc_qk = make_idesc_f16(fmt, 0, 0, 128, 128);
        const uint32_t idesc_pv = make_idesc_f16(fmt, 0, 1, 128, D);
        // One thread issues every MMA, so the issue path is kept short: descriptors of the tile
        // origins are built once, each MMA only adds a constant to them.
        const uint64_t dq0 = make_smem_desc_sw128(smem_u32(sQ), 16, 1024);
        const uint64_t dk0 = make_smem_desc_sw128(smem_u32(sKV), 16, 1024);
        const uint64_t dv0 = make_smem_desc_sw128(smem_u32(sKV), 16384, 1024);
        auto issue_qk = [&](int t, int slot) {
          const uint64_t dq = desc_advance(dq0, t * C::kHalves * 16384);
          const uint64_t dk = desc_advance(dk0, slot * C::kSlotBytes);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_f16(tmem_base + t * 128, desc_advance(dq, h * 16384 + k * 32),
                         desc_advance(dk, h * 16384 + k * 32), idesc_qk, (h | k) != 0 ? 1u : 0u);
          tc_commit(&bars->s_full[t]);
        };
        // O_t += P_t V_j in four quarters of the key range: the first MMAs start as soon as the
        // softmax warps have written P columns 0-31, while they still compute the others.
        auto issue_pv = [&](int t, int slot, int j) {
          const uint64_t dv = desc_advance(dv0, slot * C::kSlotBytes);
          const uint32_t parity = ((t == 0 ? base0 : base1) + j) & 1;
          bool got = true;
#pragma unroll
          for (int part = 0; part < 4 && got; ++part) {
            got = mbar_wait(&bars->p_half[4 * t + part], parity, p.status, kStatusTimeoutTmemFull);
            tc_fence_after();
            if (!got) break;
#pragma unroll
            for (int k = part * 2; k < part * 2 + 2; ++k)
              tc_mma_f16_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + k * 8,
                            desc_advance(dv, k * 2048), idesc_pv, (j | k) != 0 ? 1u : 0u);
          }
          if (got) tc_commit(&bars->o_done[t]);
          return got;
        };
        FwdRing<C::kSlots> at = ring;     // of the next item: K_0 V_0 K_1 V_1 ...
        auto wait_item = [&] {
          const bool got = mbar_wait(&bars->kv_full[at.slot], at.phase, p.status, kStatusTimeoutFull);
          tc_fence_after();
          return got;
        };
        bool ok = mbar_wait(&bars->q_full, units & 1, p.status, kStatusTimeoutFull) && wait_item();
        if (ok) {
          issue_qk(0, at.slot);
          if (u.n1 > 0) issue_qk(1, at.slot);
          tc_commit(&bars->kv_empty[at.slot]);
          if (n == 1) tc_commit(&bars->q_free);
          at.advance();
        }
        for (int j = 0; j < n && ok; ++j) {
          const int vslot = at.slot;
          ok = wait_item();
          if (!ok) break;
          at.advance();
          if (j < u.n0) {
            ok = issue_pv(0, vslot, j);
            if (!ok) break;
          }
          const int kslot = at.slot;
          if (j + 1 < n) {
            ok = wait_item();
            if (!ok) break;
            at.advance();
          }
          if (j + 1 < u.n0) issue_qk(0, kslot);
          if (j < u.n1) {
            ok = issue_pv(1, vslot, j);
            if (!ok) break;
          }
          tc_commit(&bars->kv_empty[vslot]);
          if (j + 1 < u.n1) issue_qk(1, kslot);
          if (j + 1 < n) tc_commit(&bars->kv_empty[kslot]);
          if (j + 2 == n) tc_commit(&bars->q_free);
        }
        if (!ok) give_up(&bars->gave_up);
      }
      __syncwarp();
      // every lane tracks the ring position, whichever lane is elected next time
      ring.phase ^= static_cast<uint32_t>(((ring.slot + 2 * n) / C::kSlots) & 1);
      ring.slot = (ring.slot + 2 * n) % C::kSlots;
      ++units;
      base0 += u.n0;
      base1 += u.n1;
    });
  } else {
    int base = 0;                        // key tiles that this warpgroup's query tile has met
    each_block([&](int, int block) {
      if (block >= work) {
        const int part = block - work, parts = gridDim.x - work, tid = threadIdx.x - 64;
        clear_rows<D>(p.o, p.o_strides[0], p.o_strides[1], p.used, p.rows, p.heads, part, parts, tid, 256);
        const int64_t spare = p.rows - p.used;
        for (int64_t i = part * 256 + tid; i < spare * p.heads; i += parts * 256)
          p.lse[i / spare * p.rows + p.used + i % spare] = 0.f;
        return;
      }
      // ---------------------------------------------------------------- softmax + epilogue
      const int t = (warp - 2) >> 2;       // query tile of this warpgroup
      const int quarter = warp & 3;        // TMEM lane quarter
      const int r_local = quarter * 32 + lane;
      int qt, nt, len;
      {   // only this lives through the loop; the rest is worked out again for the stores
        const FwdUnit<kPair> u(p, block);
        qt = t == 0 ? u.qt0 : u.qt1;
        nt = t == 0 ? u.n0 : u.n1;
        len = u.w.len;
      }
      const uint32_t lane_bits = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_addr = tmem_base + t * 128 + lane_bits;
      const uint32_t o_addr = tmem_base + 256 + t * 128 + lane_bits;
      const float sl2 = p.scale * kLog2e;
      float m_run = -INFINITY, l_run = 0.f;
      bool ok = true;
      for (int j = 0; j < nt && ok; ++j) {
        ok = warp_wait(&bars->s_full[t], (base + j) & 1, p.status, kStatusTimeoutTmemFull);
        if (!ok) break;
        tc_fence_after();
        const bool diag = p.causal && (j == qt);
        const bool tail = (j + 1) * kTile > len;
        const int col_limit_tail = len - j * kTile;  // valid columns in a tail tile
        // One TMEM read of the whole 128-column score row: the four loads are issued back to back
        // and waited for once, so their latency overlaps.
        uint32_t r[4][32];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, r[c]);
        tmem_ld_wait();
        if (diag || tail) {   // rare: the diagonal tile of a causal row block, or a ragged last tile
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int col = c * 32 + i;
              if ((diag && col > r_local) || (tail && col >= col_limit_tail)) r[c][i] = 0xff800000u;  // -inf
            }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          mx0 = fmaxf(mx0, __uint_as_float(r[0][i]));
          mx1 = fmaxf(mx1, __uint_as_float(r[1][i]));
          mx2 = fmaxf(mx2, __uint_as_float(r[2][i]));
          mx3 = fmaxf(mx3, __uint_as_float(r[3][i]));
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
        const float m_new = fmaxf(m_run, mx * sl2);
        if (j == 0) {
          m_run = m_new;
        } else {
          const bool need = m_new > m_run + kRescaleThreshold;
          if (__any_sync(0xffffffffu, need)) {
            const float m_upd = need ? m_new : m_run;
            const float alpha = exp2f(m_run - m_upd);
            l_run *= alpha;
            m_run = m_upd;
            // PV_{j-1} must have landed before O is touched
            ok = warp_wait(&bars->o_done[t], (base + j - 1) & 1, p.status, kStatusTimeoutTmemFull);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o16[16];
              tmem_ld_32x32b_x16(o_addr + c * 16, o16);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o16[i] = __float_as_uint(__uint_as_float(o16[i]) * alpha);
              tmem_st_32x32b_x16(o_addr + c * 16, o16);
            }
            tmem_st_wait();
          }
        }
        // P = exp2(s * scale_log2 - m), packed to 16 bit into the first 64 score columns
        float ls0 = 0.f, ls1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p0 = exp2f(fmaf(__uint_as_float(r[c][2 * i]), sl2, -m_run));
            const float p1 = exp2f(fmaf(__uint_as_float(r[c][2 * i + 1]), sl2, -m_run));
            ls0 += p0;
            ls1 += p1;
            pk[i] = pack_pair(p0, p1, DT);
          }
          tmem_st_32x32b_x16(s_addr + c * 16, pk);
          {   // a quarter of the key range is complete: hand it to the MMA warp
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_half[4 * t + c]);
          }
        }
        const float lsum = ls0 + ls1;
        l_run += lsum;
      }
      if (ok && nt > 0) {
        ok = warp_wait(&bars->o_done[t], (base + nt - 1) & 1, p.status, kStatusTimeoutTmemFull);
        tc_fence_after();
      }
      if (ok && nt > 0) {
        asm volatile("" : "+r"(block));
        const FwdUnit<kPair> u(p, block);
        const PackedTile& w = u.w;
        const int head = kPair ? u.head0 + t : u.head0;
        const float inv_l = 1.0f / l_run;
        const int q_local = qt * kTile + r_local;      // row inside the document
        const bool row_ok = q_local < w.len;
        const int64_t q_row = static_cast<int64_t>(w.start) + q_local;
        uint16_t* rows = reinterpret_cast<uint16_t*>(p.o) + (static_cast<int64_t>(w.start) + qt * kTile) * p.o_strides[0] +
                         head * p.o_strides[1];
        if (p.residue == nullptr) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32)
            store_columns<DT>(o_addr, c, rows, p.o_strides[0], quarter * 32, w.len - qt * kTile, inv_l, lane);
        } else {   // a training step: its backward takes rowsum(dO * O) from the unrounded O
          uint16_t* left = reinterpret_cast<uint16_t*>(p.residue) +
                           ((static_cast<int64_t>(w.start) + qt * kTile) * p.heads + head) * D;
          store_with_residue<D, DT>(o_addr, rows, p.o_strides[0], left, static_cast<int64_t>(p.heads) * D, quarter * 32,
                                    w.len - qt * kTile, inv_l, lane);
        }
        if (row_ok)
          p.lse[static_cast<int64_t>(head) * p.rows + q_row] = (m_run + log2f(l_run)) * kLn2;
      }
      if (!ok) give_up(&bars->gave_up);
      base += nt;
    });
    // A unit ends without a CTA-wide barrier: the next unit's loads and first score MMAs overlap the
    // stores of this one. Its first O += P V MMAs, which overwrite the accumulators, wait for its first P,
    // and a softmax warp writes that only after it has read its part of these accumulators.
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, int DT, bool kPair>
cudaError_t launch_fwd(const PackedAttnArgs& a, cudaStream_t st) {
  using C = FwdCfg<D>;
  CUtensorMap tq, tk, tv;
  ETHB_TRY(make_tmap_rhd(&tq, a.q, a.dtype, D, a.rows, a.heads, a.q_strides), "packed forward: q");
  ETHB_TRY(make_tmap_rhd(&tk, a.k, a.dtype, D, a.rows, a.kv_heads, a.k_strides), "packed forward: k");
  ETHB_TRY(make_tmap_rhd(&tv, a.v, a.dtype, D, a.rows, a.kv_heads, a.v_strides), "packed forward: v");
  static std::atomic<uint64_t> done{0};
  ETHB_TRY(allow_smem(packed_fwd_kernel<D, DT, kPair>, C::kSmemBytes, done), "packed forward: shared memory");
  const int units = kPair ? a.heads / 2 : a.heads;
  // a few more CTAs clear the rows behind the last document
  const int64_t spare = static_cast<int64_t>(a.rows - a.used) * a.heads * (D / 8);
  const int clear = static_cast<int>(spare == 0 ? 0 : spare < 148 * 2560 ? (spare + 2559) / 2560 : 148);
  const int64_t grid = static_cast<int64_t>(a.num_tiles) * units + clear;
  ETHB_RETURN_IF(grid > 0x7fffffff, cudaErrorInvalidValue, "packed forward: too many tiles for one grid");
  if (grid == 0) return cudaSuccess;
  packed_fwd_kernel<D, DT, kPair><<<static_cast<unsigned>(grid), C::kThreads, C::kSmemBytes, st>>>(tq, tk, tv, a);
  count_launch();
  return cudaGetLastError();
}

// ==============================================================================================
// backward
// ==============================================================================================
// dK / dV: one unit of work per (key tile, key/value head); it streams the query tiles that see the
// tile, for every head of the group in turn, so the gradients of shared heads are summed in the
// accumulators in a fixed order. dQ: one unit per (query tile, head). Both recompute the scores.
//
// Both kernels keep two 128-row tiles resident and stream pairs of tiles through a ring of five 32 KB
// slots; score and gradient tiles are 128 x 128, one buffer each:
//   S [0,128)   dP [128,256)   accumulators from column 256 on.
// Each of the two softmax warpgroups works on 64 of the 128 columns, one thread per row. Its 16-bit P
// (dS) goes over the first half of the S (dP) columns that it has read itself. With one buffer each,
// what overlaps is the two halves of an iteration: while the exponentials of S are taken the tensor
// core works on the dP side, and the other way round. (64-column tiles with two buffers of S and dP,
// as in attention_sm100.cu, need 1.25 times the shared-memory reads per MMA and leave the tensor core
// waiting for the softmax of a buffer: 133 and 107 us for dK / dV and dQ at 8192 rows of nine documents, 16
// heads of 128; now 109 and 80 us = 47 and 51 % of the tensor pipe's cycles. What bounds them is the chain
// "P written -> dV += P^T dO -> next S -> its exponentials"; a second S buffer does not fit beside two
// accumulators of 128 columns in 512 TMEM columns. With D = 64 it would; that has not been tried.)
template <int D> struct BwdCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kHalves * 16384;        // one 128-row tile
  static constexpr int kSlots = 5;
  // [lse | delta of two query tiles, 2 KB][barriers, 1 KB][two resident tiles][ring]: with D = 128 all
  // 227 KB that a block may have, so the tiles rely on the 1024-byte alignment of dynamic shared memory
  static constexpr int kFrontBytes = 3 * 1024;
  static constexpr int kSmemBytes = kFrontBytes + (2 + kSlots) * kTileBytes;
  static constexpr int kThreads = 320;
};

struct BwdBarriers {
  uint64_t res_full;
  uint64_t tail_full;     // both streamed tiles at a document's end have landed, rows behind the end not yet cleared
  uint64_t full[5];
  uint64_t empty[5];
  uint64_t s_full;        // S of an iteration is complete
  uint64_t dp_full;       // dP of an iteration is complete
  uint64_t s_read;        // dK / dV: P is written; dQ: S has been read
  uint64_t ds_half;       // dQ: the first 32 of each warpgroup's 64 dS columns are written
  uint64_t ds_full;       // dS is written
  uint64_t done;
  uint64_t kv_free;       // dK / dV: the last score MMAs of a unit have read K and V
  uint64_t qdo_full;      // dQ: the Q and dO rows of the tile sit in TMEM
  uint64_t unit_full[2];  // the next unit of work is known
  uint64_t unit_empty[2];
  int unit[2];
  uint32_t tmem_base;
  int gave_up;            // see Marks
};

// Position in the ring of slots.
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int by) {   // by < 5
    slot += by;
    if (slot >= 5) { slot -= 5; phase ^= 1; }
  }
  __device__ __forceinline__ RingPos next(int by) const {
    RingPos r = *this;
    r.advance(by);
    return r;
  }
};

// Barriers, TMEM and tensor maps of a backward CTA; false if shared memory is not laid out as assumed.
__device__ __forceinline__ bool bwd_setup(uint8_t* smem, BwdBarriers* bars, int warp, const CUtensorMap& tq,
                                          const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                                          int* status) {
  if ((smem_u32(smem) & 1023) != 0) {
    if (threadIdx.x == 0 && status != nullptr) atomicCAS(status, 0, kStatusBadArgument);
    return false;
  }
  if (threadIdx.x == 0) {
    bars->gave_up = 0;
    mbar_init(&bars->res_full, 1);
    mbar_init(&bars->tail_full, 2);
    for (int s = 0; s < 5; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->dp_full, 1);
    mbar_init(&bars->s_read, 8);      // one arrival per softmax warp
    mbar_init(&bars->ds_half, 8);
    mbar_init(&bars->ds_full, 8);
    mbar_init(&bars->done, 1);
    mbar_init(&bars->kv_free, 1);
    mbar_init(&bars->qdo_full, 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->unit_full[s], 1);
      mbar_init(&bars->unit_empty[s], 9);   // every warp but the producer's
    }
    fence_mbar_init();
    prefetch_tmap(&tq); prefetch_tmap(&tk); prefetch_tmap(&tv); prefetch_tmap(&tdo);
  }
  if (warp == 1) tmem_alloc(&bars->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return true;
}

// The three backward kernels are launched so that each may start while the one before it ends: dK / dV sets up and
// loads its first tiles while the last rows of delta are summed, dQ, which needs nothing of dK / dV, fills the
// SMs whose CTAs have run out of units. dK / dV reads delta and the counters behind `after_prerequisite`; it
// lets dQ start behind that, so delta is complete for dQ too; dQ ends only after dK / dV has.
// Forward and backward, replayed: 40 documents of 4001 tokens, 16 / 2 heads of 64, 82 us without, 77 with; nine
// documents, 8192 rows, 16 heads of 128, 340 and 335; 32 / 8 heads 863 and 857.
__device__ __forceinline__ void after_prerequisite() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The unit of work that this CTA takes as its `it`-th, -1 when there is none left. Units are sorted
// heaviest first and taken from a common counter, so CTAs with short units take more of them: which CTA
// works on a unit depends on timing, its result does not. The producer warp asks (its loads run ahead,
// so the answer is there before the others need it) and passes the number on.
__device__ __forceinline__ int next_unit(BwdBarriers* bars, int it, int units, int* counter, int warp, int lane,
                                         const Marks& marks) {
  const int b = it & 1;
  const uint32_t phase = static_cast<uint32_t>(it >> 1) & 1;
  int unit = -1;
  if (warp == 0) {
    if (lane == 0) unit = it == 0 ? static_cast<int>(blockIdx.x) : static_cast<int>(gridDim.x) + atomicAdd(counter, 1);
    unit = __shfl_sync(0xffffffffu, unit, 0);
    if (unit >= units) unit = -1;
    if (!warp_wait(&bars->unit_empty[b], phase ^ 1, marks, kStatusTimeoutEmpty)) unit = -1;
    if (lane == 0) {
      bars->unit[b] = unit;
      mbar_arrive(&bars->unit_full[b]);
    }
    __syncwarp();
    return unit;
  }
  if (!warp_wait(&bars->unit_full[b], phase, marks, kStatusTimeoutFull)) return -1;
  unit = *reinterpret_cast<volatile int*>(&bars->unit[b]);
  __syncwarp();
  if (lane == 0) mbar_arrive(&bars->unit_empty[b]);
  return unit;
}

// Producer warp: streams tile `row` of two tensors (heads ha, hb) through the next two slots. With
// tail_rows < 128 the tile ends its document: the rows behind are summands of the accumulators and are
// cleared before the slots are handed on, as 0 times what stands there may be NaN.
template <int D>
__device__ __forceinline__ bool stream_pair(BwdBarriers* bars, uint8_t* ring, RingPos& pos, uint32_t& cuts,
                                            const CUtensorMap* ma, const CUtensorMap* mb, int row, int head,
                                            int tail_rows, int lane, const Marks& marks) {
  using C = BwdCfg<D>;
  const bool cut = tail_rows < kTile;
  const int first = pos.slot;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    if (!warp_wait(&bars->empty[pos.slot], pos.phase ^ 1, marks, kStatusTimeoutEmpty)) return false;
    if (elect_one()) {
      uint64_t* full = cut ? &bars->tail_full : &bars->full[pos.slot];
      mbar_expect_tx(full, C::kTileBytes);
#pragma unroll
      for (int h = 0; h < C::kHalves; ++h)
        tma_load_3d(ring + pos.slot * C::kTileBytes + h * 16384, a == 0 ? ma : mb, full, h * 64, row, head);
    }
    __syncwarp();
    pos.advance(1);
  }
  if (cut) {
    const int second = first == 4 ? 0 : first + 1;
    if (!warp_wait(&bars->tail_full, cuts & 1, marks, kStatusTimeoutFull)) return false;
    ++cuts;
    clear_tail<C::kHalves>(ring + first * C::kTileBytes, tail_rows, lane);
    clear_tail<C::kHalves>(ring + second * C::kTileBytes, tail_rows, lane);
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&bars->full[first]);
      mbar_arrive(&bars->full[second]);
    }
  }
  return true;
}

// Barrier of a warpgroup that also tells all of it whether everybody is still `ok`.
__device__ __forceinline__ bool wg_and(int wg, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.cta.red.and.pred q, %2, 128, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "r"(wg + 1)
      : "memory");
  return all != 0;
}

// All of a warpgroup has the same unit of work, or, where a wait gave up in one of its warps, none.
__device__ __forceinline__ int wg_unit(int wg, int v) { return wg_and(wg, v >= 0) ? v : -1; }

// A wait of this CTA gave up: stop after this tile. A warpgroup decides together, its barrier needs all of it.
__device__ __forceinline__ bool go_on(int warp, const Marks& marks) {
  const bool go = *reinterpret_cast<const volatile int*>(marks.gave_up) == 0;
  return warp < 2 ? __all_sync(0xffffffffu, go) : wg_and((warp - 2) >> 2, go);
}

// delta[h, row] = sum_d dO * O, with the residue of O where the forward left one: the rounding of O to 16
// bits would otherwise be a common error of a row's whole dS (dQ and dK of 8192 rows in nine documents: 1.5
// times the error of the formula with only its results rounded, against 1.45). A (row, head) vector of
// head_dim elements is covered by head_dim / 8 adjacent lanes with one 16-byte load each per tensor (head_dim
// is 64 or 128: 8 or 16 lanes); a
// thread takes kDeltaRows of them, strided by the grid, and issues all their loads before any
// arithmetic, so 2 * kDeltaRows requests are in flight per thread. The gradients of rows that belong
// to no document are cleared here as well.
constexpr int kDeltaRows = 4;
template <int D, typename Index>   // Index: 32 bits where they hold rows x heads, the divisions are the work here
__global__ void __launch_bounds__(256) packed_delta_kernel(const PackedAttnArgs p) {
  allow_dependents();
  constexpr int lanes = D / 8;
  const Index heads = static_cast<Index>(p.heads);
  constexpr int rows_per_block = 256 / lanes;
  const int64_t total = static_cast<int64_t>(p.used) * p.heads;
  const int sub = threadIdx.x / lanes, vec = threadIdx.x % lanes;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * rows_per_block;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_block + sub;
  uint4 ov[kDeltaRows], lv[kDeltaRows], gv[kDeltaRows];
#pragma unroll
  for (int u = 0; u < kDeltaRows; ++u) {
    const int64_t i = row0 + u * stride;
    if (i < total) {
      const Index n = static_cast<Index>(i);
      const int h = static_cast<int>(n % heads);
      const int64_t s = n / heads;
      ov[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.o) + s * p.o_strides[0] +
                                              h * p.o_strides[1] + vec * 8);
      gv[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.d_o) + s * p.do_strides[0] +
                                              h * p.do_strides[1] + vec * 8);
      lv[u] = p.residue == nullptr
                  ? make_uint4(0, 0, 0, 0)
                  : reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.residue) + i * D)[vec];
    } else {
      ov[u] = make_uint4(0, 0, 0, 0);
      lv[u] = make_uint4(0, 0, 0, 0);
      gv[u] = make_uint4(0, 0, 0, 0);
    }
  }
#pragma unroll
  for (int u = 0; u < kDeltaRows; ++u) {
    const uint32_t ow[4] = {ov[u].x, ov[u].y, ov[u].z, ov[u].w}, gw[4] = {gv[u].x, gv[u].y, gv[u].z, gv[u].w};
    const uint32_t lw[4] = {lv[u].x, lv[u].y, lv[u].z, lv[u].w};
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = unpack2(ow[e], p.dtype), l = unpack2(lw[e], p.dtype), d = unpack2(gw[e], p.dtype);
      acc += (a.x + l.x) * d.x + (a.y + l.y) * d.y;
    }
#pragma unroll
    for (int off = lanes >> 1; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    const int64_t i = row0 + u * stride;
    if (vec == 0 && i < total) {
      const Index n = static_cast<Index>(i);
      p.delta[static_cast<int64_t>(n % heads) * p.rows + static_cast<int64_t>(n / heads)] = acc;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < 2) p.counters[threadIdx.x] = 0;   // of the two kernels that follow
  if (p.used < p.rows) {
    clear_rows<D>(p.dq, p.dq_strides[0], p.dq_strides[1], p.used, p.rows, p.heads, blockIdx.x, gridDim.x, threadIdx.x, 256);
    clear_rows<D>(p.dk, p.dk_strides[0], p.dk_strides[1], p.used, p.rows, p.kv_heads, blockIdx.x, gridDim.x, threadIdx.x, 256);
    clear_rows<D>(p.dv, p.dv_strides[0], p.dv_strides[1], p.used, p.rows, p.kv_heads, blockIdx.x, gridDim.x, threadIdx.x, 256);
  }
}

// dV | dK = sum over the splits, in their order: one thread per eight columns.
template <int D>
__global__ void __launch_bounds__(256) packed_join_kernel(const PackedAttnArgs p) {
  constexpr int kChunks = D / 8;
  const int64_t per = static_cast<int64_t>(p.used) * p.kv_heads * kChunks;      // chunks of one tensor
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= 2 * per) return;
  const int which = at >= per;                                                 // 0: dV, 1: dK
  const int64_t i = at - which * per;
  float sum[8] = {};
  for (int sp = 0; sp < p.splits; ++sp) {
    const float4* src = reinterpret_cast<const float4*>(p.parts + ((sp * 2 + which) * per + i) * 8);
    const float4 a = src[0], b = src[1];
    sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
    sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
  }
  const int c = static_cast<int>(i % kChunks);
  const int64_t rh = i / kChunks, row = rh / p.kv_heads, head = rh % p.kv_heads;
  uint16_t* dst = which == 0 ? reinterpret_cast<uint16_t*>(p.dv) + row * p.dv_strides[0] + head * p.dv_strides[1]
                             : reinterpret_cast<uint16_t*>(p.dk) + row * p.dk_strides[0] + head * p.dk_strides[1];
  reinterpret_cast<uint4*>(dst)[c] = make_uint4(pack2(sum[0], sum[1], p.dtype), pack2(sum[2], sum[3], p.dtype),
                                                pack2(sum[4], sum[5], p.dtype), pack2(sum[6], sum[7], p.dtype));
}

// ---- dK / dV: persistent CTAs over (key/value tile, key/value head) ------------------------------
// One CTA per SM takes units of work from a list sorted heaviest first (under the causal mask key tile j
// meets tiles - j query tiles of each head). Where heads share a key/value head and there are too few
// units for the SMs, a unit is split by heads (`splits`, see attention_packed_splits) and packed_join_kernel
// adds the parts.
// TMEM, the barriers and the tensor-map prefetch are set up once per CTA; barrier parities therefore
// run on counters that persist across tiles (`it`: units done by this CTA, `g`: query tiles streamed).
// No CTA-wide barrier separates the tiles: the loads and first score MMAs of the next tile overlap the
// accumulator stores of the current one.
//
// S^T = K Q^T and dP^T = V dO^T, so P^T and dS^T are A operands of dV += P^T dO and dK += dS^T Q.
// The tensor core's order is  dV(i) S(i+1) | dK(i) dP(i+1):  the first pair needs P(i), the second dS(i).
template <int D, int DT>
__global__ void __launch_bounds__(320, 1)
packed_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                       const PackedAttnArgs p) {
  using C = BwdCfg<D>;
  extern __shared__ uint8_t smem[];
  float* sAux = reinterpret_cast<float*>(smem);
  BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + 2048);
  uint8_t* sK = smem + C::kFrontBytes;
  uint8_t* sV = sK + C::kTileBytes;
  uint8_t* sRing = sV + C::kTileBytes;          // Q_0 dO_0 Q_1 dO_1 ...

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.kv_heads, share = group / p.splits;
  const int units = p.num_k_tiles * p.kv_heads * p.splits;
  if (!bwd_setup(smem, bars, warp, tq, tk, tv, tdo, p.status)) return;
  const Marks marks{p.status, &bars->gave_up};
  const uint32_t tmem_base = bars->tmem_base;
  RingPos pos;               // producer and MMA issuer: slot of the next Q tile
  uint32_t cuts = 0;         // producer: tile pairs at a document's end so far
  int g = 0;                 // query tiles streamed by this CTA before the current tile

  const auto next = [&](int it) {
    const int unit = next_unit(bars, it, units, p.counters, warp, lane, marks);
    return warp < 2 ? unit : wg_unit((warp - 2) >> 2, unit);
  };
  const auto tile_of = [&](int unit) { return p.k_tiles[unit / (p.kv_heads * p.splits)]; };
  int unit = next(0), unit_next = -1;
  PackedTile w_next{};
  float next_lse = INFINITY, next_delta = 0.f;   // softmax: of the next query tile, requested ahead
  if (warp >= 2) {
    after_prerequisite();
    if (warp == 2) allow_dependents();
  }
  if (unit >= 0) w_next = tile_of(unit);
  for (int it = 0; unit >= 0; ++it, unit = unit_next) {
    const PackedTile w = w_next;
    const int kv_head = unit % (p.kv_heads * p.splits) / p.splits, part = unit % p.splits;
    const int head0 = kv_head * group + part * share;
    const int j = w.tile;                          // key/value tile inside the document
    const int q_tiles = (w.len + kTile - 1) / kTile;
    const int i0 = p.causal ? j : 0;
    const int nd = q_tiles - i0;                   // query tiles of the document that see these keys
    const int nq = nd * share;                     // streamed: all of them for every head of this split
    const int last_rows = w.len - (q_tiles - 1) * kTile;   // rows of the document's last tile
    if (warp == 0) {
      bool ok = true;
      for (int t = 0, i = i0, head = head0; t < nq && ok; ++t) {
        ok = stream_pair<D>(bars, sRing, pos, cuts, &tq, &tdo, w.start + i * kTile, head,
                            i == q_tiles - 1 ? last_rows : kTile, lane, marks);
        if (++i == q_tiles) { i = i0; ++head; }
        if (t > 0) continue;
        // the resident K / V buffers are free once the last score MMAs of the previous unit are through;
        // its last softmax, gradient MMAs and stores then overlap these loads
        ok = ok && (it == 0 || warp_wait(&bars->kv_free, (it - 1) & 1, marks, kStatusTimeoutTmemFull));
        if (ok && elect_one()) {
          mbar_expect_tx(&bars->res_full, 2 * C::kTileBytes);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h) {
            tma_load_3d(sK + h * 16384, &tk, &bars->res_full, h * 64, w.start + j * kTile, kv_head);
            tma_load_3d(sV + h * 16384, &tv, &bars->res_full, h * 64, w.start + j * kTile, kv_head);
          }
        }
        __syncwarp();
      }
      if (it == 0) after_prerequisite();       // the counter is cleared
      unit_next = next(it + 1);
      if (unit_next >= 0) w_next = tile_of(unit_next);
    } else if (warp == 1) {
      if (elect_one()) {
        const int fmt = DT == kBF16 ? 1 : 0;
        const uint32_t idesc_s = make_idesc_f16(fmt, 0, 0, 128, 128);
        const uint32_t idesc_acc = make_idesc_f16(fmt, 0, 1, 128, D);
        // One thread issues every MMA, so the issue path is kept short: descriptors of the tile
        // origins are built once, each MMA only adds a constant to them.
        const uint64_t dK0 = make_smem_desc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t dV0 = make_smem_desc_sw128(smem_u32(sV), 16, 1024);
        const uint64_t dRk = make_smem_desc_sw128(smem_u32(sRing), 16, 1024);          // K-major view
        const uint64_t dRm = make_smem_desc_sw128(smem_u32(sRing), 16384, 1024);       // MN-major view
        auto issue_scores = [&](uint64_t a0, int slot, uint32_t tmem, uint64_t* full) {
          const uint64_t b0 = desc_advance(dRk, slot * C::kTileBytes);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_f16(tmem_base + tmem, desc_advance(a0, h * 16384 + k * 32),
                         desc_advance(b0, h * 16384 + k * 32), idesc_s, (h | k) != 0 ? 1u : 0u);
          tc_commit(full);
        };
        // queries 0-63 of P / dS sit at columns [0, 32) of their buffer, queries 64-127 at [64, 96)
        auto issue_acc = [&](uint32_t acc, uint32_t a, int slot, bool first) {
          const uint64_t b0 = desc_advance(dRm, slot * C::kTileBytes);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc_mma_f16_ts(tmem_base + acc, tmem_base + a + (k >> 2) * 64 + (k & 3) * 8, desc_advance(b0, k * 2048),
                          idesc_acc, first && k == 0 ? 0u : 1u);
          tc_commit(&bars->empty[slot]);
        };
        auto wait_full = [&](const RingPos& at) {
          const bool got = marked_wait(&bars->full[at.slot], at.phase, marks, kStatusTimeoutFull);
          tc_fence_after();
          return got;
        };
        auto wait_softmax = [&](uint64_t* bar, int iter) {
          const bool got = marked_wait(bar, iter & 1, marks, kStatusTimeoutTmemFull);
          tc_fence_after();
          return got;
        };
        RingPos at = pos;
        bool ok = marked_wait(&bars->res_full, it & 1, marks, kStatusTimeoutFull) && wait_full(at);
        if (ok) {
          issue_scores(dK0, at.slot, 0, &bars->s_full);
          ok = wait_full(at.next(1));
          if (ok) issue_scores(dV0, at.next(1).slot, 128, &bars->dp_full);
          if (nq == 1) tc_commit(&bars->kv_free);
        }
        for (int t = 0; t < nq && ok; ++t) {
          const RingPos qi = at, doi = at.next(1), qn = at.next(2), don = at.next(3);
          ok = wait_softmax(&bars->s_read, g + t);
          if (!ok) break;
          issue_acc(256, 0, doi.slot, t == 0);                     // dV += P^T dO
          if (t + 1 < nq) {
            ok = wait_full(qn);
            if (!ok) break;
            issue_scores(dK0, qn.slot, 0, &bars->s_full);
          }
          ok = wait_softmax(&bars->ds_full, g + t);
          if (!ok) break;
          issue_acc(384, 128, qi.slot, t == 0);                    // dK += dS^T Q
          if (t + 1 < nq) {
            ok = wait_full(don);
            if (!ok) break;
            issue_scores(dV0, don.slot, 128, &bars->dp_full);
            if (t + 2 == nq) tc_commit(&bars->kv_free);
          }
          at = qn;
        }
        tc_commit(&bars->done);
      }
      __syncwarp();
      // every lane tracks the ring position, whichever lane is elected next time
      const int items = 2 * nq;
      pos.phase ^= static_cast<uint32_t>(((pos.slot + items) / 5) & 1);
      pos.slot = (pos.slot + items) % 5;
      unit_next = next(it + 1);
      if (unit_next >= 0) w_next = tile_of(unit_next);
    } else {
      const int wg = (warp - 2) >> 2;      // columns [64 wg, 64 wg + 64) of every tile
      const int quarter = warp & 3;
      const int r_local = quarter * 32 + lane;     // key/value row inside the tile
      const int wg_tid = threadIdx.x - 64 - wg * 128;
      const uint32_t lane_bits = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_addr = tmem_base + wg * 64 + lane_bits, dp_addr = s_addr + 128;
      const float sl2 = p.scale * kLog2e;
      bool ok = true;
      // -lse / -delta of this warpgroup's 64 queries, staged one query tile ahead: the global loads for
      // tile t + 1 are issued before tile t is processed and parked in shared memory after it, so their
      // latency is never waited for. Streamed tile t is query tile i0 + t % nd of head head0 + t / nd.
      auto aux_load = [&](const PackedTile& doc, int i, int head, float& lse, float& delta) {
        const int qi = i * kTile + wg * 64 + wg_tid;
        const bool in = qi < doc.len;
        const int64_t at = static_cast<int64_t>(head) * p.rows + doc.start + qi;
        lse = in ? -p.lse[at] * kLog2e : -INFINITY;
        delta = in ? -p.delta[at] : 0.f;
      };
      auto aux_slot = [&](int t) { return sAux + ((wg * 2 + (t & 1)) * 2) * 64; };   // [lse 64 | delta 64]
      if (it == 0 && wg_tid < 64) aux_load(w, i0, head0, next_lse, next_delta);
      if (wg_tid < 64) {   // everyone has left the previous unit's tiles: `next` has a barrier
        aux_slot(0)[wg_tid] = next_lse;
        aux_slot(0)[64 + wg_tid] = next_delta;
      }
      int i = i0, head = head0;
      for (int t = 0; t < nq; ++t) {
        const int i_next = i + 1 == q_tiles ? i0 : i + 1, head_next = i + 1 == q_tiles ? head + 1 : head;
        ok = wg_and(wg, ok);             // tile t's values are staged; everyone has left tile t - 1
        if (!ok) break;
        if (wg_tid < 64 && t + 1 < nq) aux_load(w, i_next, head_next, next_lse, next_delta);
        const bool diag = p.causal && (i == j);
        const float* a_lse = aux_slot(t);
        const float* a_del = a_lse + 64;
        Pair pv[32];
        ok = warp_wait(&bars->s_full, (g + t) & 1, marks, kStatusTimeoutTmemFull);
        if (!ok) continue;
        tc_fence_after();
        {
          uint32_t rs[2][32];
          tmem_ld_32x32b_x32(s_addr, rs[0]);
          tmem_ld_32x32b_x32(s_addr + 32, rs[1]);
          tmem_ld_wait();
          const Pair scale = pair(sl2, sl2);
          // -lse comes as 16-byte broadcast loads (four query columns each); only the tile on the
          // diagonal pays for the causal mask
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const float4 l4 = *reinterpret_cast<const float4*>(a_lse + 4 * y);
            const uint32_t* r4 = &rs[y >> 3][(4 * y) & 31];
            pv[2 * y] = exp2_mixed<kBwdPoly>(
                2 * y, fma2(pair(__uint_as_float(r4[0]), __uint_as_float(r4[1])), scale, pair(l4.x, l4.y)));
            pv[2 * y + 1] = exp2_mixed<kBwdPoly>(
                2 * y + 1, fma2(pair(__uint_as_float(r4[2]), __uint_as_float(r4[3])), scale, pair(l4.z, l4.w)));
          }
        }
        if (diag) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float a, b;
            split(pv[e], a, b);
            pv[e] = pair(r_local > wg * 64 + 2 * e ? 0.f : a, r_local > wg * 64 + 2 * e + 1 ? 0.f : b);
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) pk[x] = pack_pair(pv[half * 16 + x], DT);
          tmem_st_32x32b_x16(s_addr + half * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->s_read);
        ok = warp_wait(&bars->dp_full, (g + t) & 1, marks, kStatusTimeoutTmemFull);
        if (!ok) continue;
        tc_fence_after();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t rd[32], dk[16];
          tmem_ld_32x32b_x32(dp_addr + half * 32, rd);
          tmem_ld_wait();
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const float4 e4 = *reinterpret_cast<const float4*>(a_del + half * 32 + 4 * y);
            dk[2 * y] = pack_pair(pv[half * 16 + 2 * y] * (pair(__uint_as_float(rd[4 * y]), __uint_as_float(rd[4 * y + 1])) +
                                                           pair(e4.x, e4.y)), DT);
            dk[2 * y + 1] = pack_pair(pv[half * 16 + 2 * y + 1] *
                                          (pair(__uint_as_float(rd[4 * y + 2]), __uint_as_float(rd[4 * y + 3])) +
                                           pair(e4.z, e4.w)), DT);
          }
          tmem_st_32x32b_x16(dp_addr + half * 16, dk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ds_full);
        if (wg_tid < 64 && t + 1 < nq) {
          aux_slot(t + 1)[wg_tid] = next_lse;
          aux_slot(t + 1)[64 + wg_tid] = next_delta;
        }
        i = i_next;
        head = head_next;
      }
      // what the next unit starts with is requested before this one's results are waited for and stored
      unit_next = next(it + 1);
      if (unit_next >= 0) {
        w_next = tile_of(unit_next);
        const int kv_split = unit_next % (p.kv_heads * p.splits);
        if (wg_tid < 64)
          aux_load(w_next, p.causal ? w_next.tile : 0,
                   kv_split / p.splits * group + kv_split % p.splits * share, next_lse, next_delta);
      }
      // epilogue: warpgroup 0 stores dV, warpgroup 1 stores dK * scale
      if (ok) ok = warp_wait(&bars->done, it & 1, marks, kStatusTimeoutTmemFull);
      if (ok) {
        tc_fence_after();
        // rows of the tile that exist, from its first row on
        const int valid = w.len - j * kTile, first = quarter * 32;
        const int64_t row = static_cast<int64_t>(w.start) + j * kTile;
        const uint32_t acc = tmem_base + 256 + wg * 128 + lane_bits;
        const float mul = wg == 0 ? 1.0f : p.scale;
        if (p.splits == 1) {
          const int64_t* st = wg == 0 ? p.dv_strides : p.dk_strides;
          uint16_t* rows = reinterpret_cast<uint16_t*>(wg == 0 ? p.dv : p.dk) + row * st[0] + kv_head * st[1];
#pragma unroll 1
          for (int c = 0; c < D; c += 32) store_columns<DT>(acc, c, rows, st[0], first, valid, mul, lane);
        } else {   // [split, dV | dK, row, kv_head, D] in fp32, summed by packed_join_kernel
          float* rows = p.parts + (((part * 2 + wg) * static_cast<int64_t>(p.used) + row) * p.kv_heads + kv_head) * D;
#pragma unroll 1
          for (int c = 0; c < D; c += 32)
            store_columns_f32(acc, c, rows, static_cast<int64_t>(p.kv_heads) * D, first, valid, mul, lane);
        }
      }
    }
    // End of the unit, without a CTA-wide barrier: the roles meet again only through the mbarriers. The
    // producer waits for `kv_free` before it refills K / V; the first dV / dK MMAs of the next unit
    // (which overwrite the accumulators) wait for that unit's first P, and a softmax warp writes that
    // only after it has stored its part of these accumulators.
    g += nq;
    if (!go_on(warp, marks)) break;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---- dQ: persistent CTAs over (query tile, head) -------------------------------------------------
// Like the dK / dV kernel: one CTA per SM, units heaviest first (query tile i meets i + 1 key tiles
// under the causal mask), TMEM and barriers set up once, parities on counters that persist across units
// (`it`, `g`), and no CTA-wide barrier between them: the Q / dO loads and first score MMAs of the next
// unit overlap the dQ store.
//
// S = Q K^T and dP = dO V^T read Q and dO as A operands from TMEM (columns [384, 448) and [448, 512)),
// where the softmax warps put them once per tile: an MMA then fetches only its B operand from shared
// memory. P stays in registers; only dS is written back. The tensor core's order is
// S(i+1) | dQ(i) dP(i+1):  S(i+1) needs S(i) read, the others dS(i).
template <int D, int DT>
__global__ void __launch_bounds__(320, 1)
packed_bwd_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                     const PackedAttnArgs p) {
  using C = BwdCfg<D>;
  extern __shared__ uint8_t smem[];
  BwdBarriers* bars = reinterpret_cast<BwdBarriers*>(smem + 2048);
  uint8_t* sQ = smem + C::kFrontBytes;
  uint8_t* sDO = sQ + C::kTileBytes;
  uint8_t* sRing = sDO + C::kTileBytes;         // K_0 V_0 K_1 V_1 ...

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.kv_heads;
  const int units = p.num_q_tiles * p.heads;
  if (!bwd_setup(smem, bars, warp, tq, tk, tv, tdo, p.status)) return;
  const Marks marks{p.status, &bars->gave_up};
  const uint32_t tmem_base = bars->tmem_base;
  RingPos pos;               // producer and MMA issuer: slot of the next K tile
  uint32_t cuts = 0;         // producer: tile pairs at a document's end so far
  int g = 0;                 // key/value tiles streamed by this CTA before the current tile

  const auto next = [&](int it) {
    const int unit = next_unit(bars, it, units, p.counters + 1, warp, lane, marks);
    return warp < 2 ? unit : wg_unit((warp - 2) >> 2, unit);
  };
  // Stages the rows of unit `it` as TMEM operands: warpgroup 0 copies the Q rows, warpgroup 1 the dO rows,
  // one thread per row, out of the 128-byte-swizzled tiles the TMA wrote (16-byte chunk c of row r
  // sits at chunk c ^ (r & 7)); element d of a row lands in TMEM column d / 2 of the operand. The score
  // MMAs of the unit before have been waited for.
  const auto stage_rows = [&](int it) {
    const int wg = (warp - 2) >> 2, r_local = (warp & 3) * 32 + lane;
    if (!warp_wait(&bars->res_full, it & 1, marks, kStatusTimeoutFull)) return false;
    const uint8_t* src = (wg == 0 ? sQ : sDO) + r_local * 128;
    const uint32_t dst = tmem_base + 384 + wg * 64 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll
    for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
      for (int gq = 0; gq < 2; ++gq) {
        uint32_t v[16];
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          const int c = gq * 4 + c4;
          const uint4 x = *reinterpret_cast<const uint4*>(src + h * 16384 + ((c ^ (r_local & 7)) << 4));
          v[c4 * 4 + 0] = x.x; v[c4 * 4 + 1] = x.y; v[c4 * 4 + 2] = x.z; v[c4 * 4 + 3] = x.w;
        }
        tmem_st_32x32b_x16(dst + h * 32 + gq * 16, v);
      }
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->qdo_full);
    return true;
  };
  int unit = next(0), unit_next = -1;
  PackedTile w_next{};
  float lse_next = 0.f, delta_next = 0.f;        // softmax: of this thread's row of the next unit
  const auto row_stats = [&](const PackedTile& doc, int head) {
    const int q_local = doc.tile * kTile + (warp & 3) * 32 + lane;
    const bool in = q_local < doc.len;
    const int64_t at = static_cast<int64_t>(head) * p.rows + doc.start + q_local;
    lse_next = in ? p.lse[at] : INFINITY;
    delta_next = in ? p.delta[at] : 0.f;
  };
  bool ok = true;
  if (unit >= 0) {
    w_next = p.q_tiles[unit / p.heads];
    if (warp >= 2) {
      row_stats(w_next, unit % p.heads);
      ok = stage_rows(0);
    }
  }
  for (int it = 0; unit >= 0; ++it, unit = unit_next) {
    const PackedTile w = w_next;
    const int head = unit % p.heads, kv_head = head / group;
    const int i = w.tile;                          // query tile inside the document
    const int kv_tiles = (w.len + kTile - 1) / kTile;
    const int n = p.causal ? i + 1 : kv_tiles;
    const int last_rows = w.len - (kv_tiles - 1) * kTile;   // rows of the document's last tile
    if (warp == 0) {
      // Q / dO are free once the softmax warps have copied the previous unit's rows
      ok = it == 0 || warp_wait(&bars->qdo_full, (it - 1) & 1, marks, kStatusTimeoutTmemFull);
      if (ok && elect_one()) {
        mbar_expect_tx(&bars->res_full, 2 * C::kTileBytes);
#pragma unroll
        for (int h = 0; h < C::kHalves; ++h) {
          tma_load_3d(sQ + h * 16384, &tq, &bars->res_full, h * 64, w.start + i * kTile, head);
          tma_load_3d(sDO + h * 16384, &tdo, &bars->res_full, h * 64, w.start + i * kTile, head);
        }
      }
      __syncwarp();
      for (int t = 0; t < n && ok; ++t)
        ok = stream_pair<D>(bars, sRing, pos, cuts, &tk, &tv, w.start + t * kTile, kv_head,
                            t == kv_tiles - 1 ? last_rows : kTile, lane, marks);
      unit_next = next(it + 1);
      if (unit_next >= 0) w_next = p.q_tiles[unit_next / p.heads];
    } else if (warp == 1) {
      if (elect_one()) {
        const int fmt = DT == kBF16 ? 1 : 0;
        const uint32_t idesc_s = make_idesc_f16(fmt, 0, 0, 128, 128);
        const uint32_t idesc_acc = make_idesc_f16(fmt, 0, 1, 128, D);
        // short issue path: tile-origin descriptors once, constants added per MMA
        const uint64_t dRk = make_smem_desc_sw128(smem_u32(sRing), 16, 1024);          // K-major view
        const uint64_t dRm = make_smem_desc_sw128(smem_u32(sRing), 16384, 1024);       // MN-major view
        auto issue_scores = [&](uint32_t a, int slot, uint32_t tmem, uint64_t* full) {
          const uint64_t b0 = desc_advance(dRk, slot * C::kTileBytes);
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              tc_mma_f16_ts(tmem_base + tmem, tmem_base + a + (h * 4 + k) * 8, desc_advance(b0, h * 16384 + k * 32),
                            idesc_s, (h | k) != 0 ? 1u : 0u);
          tc_commit(full);
        };
        // keys 0-63 of dS sit at columns [0, 32) of the dP buffer, keys 64-127 at [64, 96); the first 32
        // keys of each warpgroup (k-steps 0 1 4 5) are handed over before the others (2 3 6 7)
        auto issue_acc = [&](int slot, int half, bool first) {
          const uint64_t b0 = desc_advance(dRm, slot * C::kTileBytes);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int k = (q >> 1) * 4 + half * 2 + (q & 1);
            tc_mma_f16_ts(tmem_base + 256, tmem_base + 128 + (k >> 2) * 64 + (k & 3) * 8, desc_advance(b0, k * 2048),
                          idesc_acc, first && half == 0 && q == 0 ? 0u : 1u);
          }
        };
        auto wait_full = [&](const RingPos& at) {
          const bool got = marked_wait(&bars->full[at.slot], at.phase, marks, kStatusTimeoutFull);
          tc_fence_after();
          return got;
        };
        auto wait_softmax = [&](uint64_t* bar, int iter) {
          const bool got = marked_wait(bar, iter & 1, marks, kStatusTimeoutTmemFull);
          tc_fence_after();
          return got;
        };
        RingPos at = pos;
        bool ok = marked_wait(&bars->qdo_full, it & 1, marks, kStatusTimeoutFull) && wait_full(at);
        if (ok) {
          tc_fence_after();
          issue_scores(384, at.slot, 0, &bars->s_full);
          ok = wait_full(at.next(1));
          if (ok) {
            issue_scores(448, at.next(1).slot, 128, &bars->dp_full);
            tc_commit(&bars->empty[at.next(1).slot]);
          }
        }
        for (int t = 0; t < n && ok; ++t) {
          const RingPos kn = at.next(2), vn = at.next(3);
          if (t + 1 < n) {
            ok = wait_full(kn) && wait_softmax(&bars->s_read, g + t);
            if (!ok) break;
            issue_scores(384, kn.slot, 0, &bars->s_full);
          }
          ok = wait_softmax(&bars->ds_half, g + t);
          if (!ok) break;
          issue_acc(at.slot, 0, t == 0);                            // dQ += dS K
          ok = wait_softmax(&bars->ds_full, g + t);
          if (!ok) break;
          issue_acc(at.slot, 1, t == 0);
          tc_commit(&bars->empty[at.slot]);
          if (t + 1 < n) {
            ok = wait_full(vn);
            if (!ok) break;
            issue_scores(448, vn.slot, 128, &bars->dp_full);
            tc_commit(&bars->empty[vn.slot]);
          }
          at = kn;
        }
        tc_commit(&bars->done);
      }
      __syncwarp();
      // every lane tracks the ring position, whichever lane is elected next time
      const int items = 2 * n;
      pos.phase ^= static_cast<uint32_t>(((pos.slot + items) / 5) & 1);
      pos.slot = (pos.slot + items) % 5;
      unit_next = next(it + 1);
      if (unit_next >= 0) w_next = p.q_tiles[unit_next / p.heads];
    } else {
      const int wg = (warp - 2) >> 2;      // columns [64 wg, 64 wg + 64) of every tile
      const int quarter = warp & 3;
      const int r_local = quarter * 32 + lane;     // query row inside the tile
      const int q_local = i * kTile + r_local;     // row inside the document
      const uint32_t lane_bits = static_cast<uint32_t>(quarter * 32) << 16;
      const uint32_t s_addr = tmem_base + wg * 64 + lane_bits, dp_addr = s_addr + 128;
      const float sl2 = p.scale * kLog2e;
      const float neg_lse = -lse_next * kLog2e, neg_delta = -delta_next;
      for (int t = 0; t < n && ok; ++t) {
        ok = warp_wait(&bars->s_full, (g + t) & 1, marks, kStatusTimeoutTmemFull);
        if (!ok) break;
        tc_fence_after();
        const int kv0 = t * kTile + wg * 64;              // first key of this warpgroup's columns
        const bool masked = (p.causal && t == i) || kv0 + 64 > w.len;
        Pair pv[32];
        {
          uint32_t rs[2][32];
          tmem_ld_32x32b_x32(s_addr, rs[0]);
          tmem_ld_32x32b_x32(s_addr + 32, rs[1]);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->s_read);
          const Pair scale = pair(sl2, sl2), bias = pair(neg_lse, neg_lse);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            pv[e] = exp2_mixed<kBwdPoly>(e, fma2(pair(__uint_as_float(rs[e >> 4][(2 * e) & 31]),
                                                          __uint_as_float(rs[e >> 4][(2 * e + 1) & 31])), scale, bias));
        }
        if (masked) {   // the common case carries no mask
          // keys this row sees: up to itself on the diagonal tile, up to the document's end on the last
          const int seen = min(p.causal && t == i ? q_local + 1 : w.len, w.len) - kv0;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float a, b;
            split(pv[e], a, b);
            pv[e] = pair(2 * e >= seen ? 0.f : a, 2 * e + 1 >= seen ? 0.f : b);
          }
        }
        ok = warp_wait(&bars->dp_full, (g + t) & 1, marks, kStatusTimeoutTmemFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t rd[32], dk[16];
          tmem_ld_32x32b_x32(dp_addr + half * 32, rd);
          tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < 16; ++x)
            dk[x] = pack_pair(pv[half * 16 + x] * (pair(__uint_as_float(rd[2 * x]), __uint_as_float(rd[2 * x + 1])) +
                                                   pair(neg_delta, neg_delta)), DT);
          tmem_st_32x32b_x16(dp_addr + half * 16, dk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(half == 0 ? &bars->ds_half : &bars->ds_full);
        }
      }
      // the next unit's rows go into TMEM before this one's result is waited for and stored, so that its
      // first score MMAs follow the last ones of this unit
      unit_next = next(it + 1);
      if (unit_next >= 0) {
        w_next = p.q_tiles[unit_next / p.heads];
        row_stats(w_next, unit_next % p.heads);
        ok = ok && stage_rows(it + 1);
      }
      const bool here = ok && warp_wait(&bars->done, it & 1, marks, kStatusTimeoutTmemFull);
      if (here) {
        tc_fence_after();
        // each warpgroup stores half of the head dimension
        uint16_t* rows = reinterpret_cast<uint16_t*>(p.dq) + (static_cast<int64_t>(w.start) + i * kTile) * p.dq_strides[0] +
                         head * p.dq_strides[1];
#pragma unroll 1
        for (int c = wg * (D / 2); c < (wg + 1) * (D / 2); c += 32)
          store_columns<DT>(tmem_base + 256 + lane_bits, c, rows, p.dq_strides[0], quarter * 32, w.len - i * kTile, p.scale,
                            lane);
      }
    }
    // End of the unit, without a CTA-wide barrier: the first dQ MMAs of the next unit (which overwrite the
    // accumulator) wait for that unit's first dS, and a softmax warp writes that only after it has
    // stored its part of this accumulator.
    g += n;
    if (!go_on(warp, marks)) break;
  }
  if (threadIdx.x == 0) after_prerequisite();   // whatever follows in the stream may rely on dK / dV as well
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Launch that may begin before the stream's previous kernel has ended (see after_prerequisite).
template <typename Kernel, typename... Args>
cudaError_t launch_early(Kernel kernel, int64_t grid, int threads, int smem, cudaStream_t st, const Args&... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int DT>
cudaError_t launch_bwd(const PackedAttnArgs& a, cudaStream_t st) {
  using C = BwdCfg<D>;
  CUtensorMap tq, tk, tv, tdo;
  ETHB_TRY(make_tmap_rhd(&tq, a.q, a.dtype, D, a.rows, a.heads, a.q_strides), "packed backward: q");
  ETHB_TRY(make_tmap_rhd(&tk, a.k, a.dtype, D, a.rows, a.kv_heads, a.k_strides), "packed backward: k");
  ETHB_TRY(make_tmap_rhd(&tv, a.v, a.dtype, D, a.rows, a.kv_heads, a.v_strides), "packed backward: v");
  ETHB_TRY(make_tmap_rhd(&tdo, a.d_o, a.dtype, D, a.rows, a.heads, a.do_strides), "packed backward: dO");
  static std::atomic<uint64_t> done_kv{0}, done_q{0};
  ETHB_TRY(allow_smem(packed_bwd_dkdv_kernel<D, DT>, C::kSmemBytes, done_kv), "packed backward: shared memory");
  ETHB_TRY(allow_smem(packed_bwd_dq_kernel<D, DT>, C::kSmemBytes, done_q), "packed backward: shared memory");
  const int64_t k_work = static_cast<int64_t>(a.num_k_tiles) * a.kv_heads * a.splits;
  const int64_t q_work = static_cast<int64_t>(a.num_q_tiles) * a.heads;
  ETHB_RETURN_IF(k_work > 0x3fffffff || q_work > 0x3fffffff, cudaErrorInvalidValue, "packed backward: too many tiles");
  const int sms = sm_count();
  const int64_t vectors = static_cast<int64_t>(a.rows) * a.heads;
  constexpr int per_block = 256 / (D / 8) * kDeltaRows;
  const unsigned delta_grid = static_cast<unsigned>((vectors + per_block - 1) / per_block);
  if (vectors < (int64_t{1} << 32)) packed_delta_kernel<D, uint32_t><<<delta_grid, 256, 0, st>>>(a);
  else packed_delta_kernel<D, uint64_t><<<delta_grid, 256, 0, st>>>(a);
  count_launch();
  if (a.used > 0) {
    ETHB_TRY(launch_early(packed_bwd_dkdv_kernel<D, DT>, k_work < sms ? k_work : sms, C::kThreads, C::kSmemBytes, st, tq, tk,
                          tv, tdo, a), "packed backward: dK / dV");
    ETHB_TRY(launch_early(packed_bwd_dq_kernel<D, DT>, q_work < sms ? q_work : sms, C::kThreads, C::kSmemBytes, st, tq, tk, tv,
                          tdo, a), "packed backward: dQ");
    count_launch(2);
    if (a.splits > 1) {
      const int64_t chunks = 2 * static_cast<int64_t>(a.used) * a.kv_heads * (D / 8);
      packed_join_kernel<D><<<static_cast<unsigned>((chunks + 255) / 256), 256, 0, st>>>(a);
      count_launch();
    }
  }
  return cudaGetLastError();
}

cudaError_t check_common(const PackedAttnArgs& a) {
  ETHB_RETURN_IF(a.dtype != kF16 && a.dtype != kBF16, cudaErrorInvalidValue, "packed attention: fp16 or bf16 only");
  ETHB_RETURN_IF(a.head_dim != 64 && a.head_dim != 128, cudaErrorInvalidValue, "packed attention: head_dim 64 or 128");
  ETHB_RETURN_IF(a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0, cudaErrorInvalidValue,
                 "packed attention: heads must be a multiple of kv_heads");
  ETHB_RETURN_IF(a.used < 0 || a.used > a.rows || a.rows > 0x7fffff00, cudaErrorInvalidValue, "packed attention: rows");
  return cudaSuccess;
}
cudaError_t check_out(const void* base, const int64_t strides[2]) {
  ETHB_RETURN_IF((reinterpret_cast<uintptr_t>(base) & 15) != 0 || strides[0] % 8 != 0 || strides[1] % 8 != 0,
                 cudaErrorMisalignedAddress, "packed attention: outputs must be 16-byte aligned");
  return cudaSuccess;
}

template <int D, int DT>
cudaError_t launch_fwd_for(const PackedAttnArgs& a, cudaStream_t st) {
  return attention_packed_pairs_heads(a.heads, a.kv_heads) ? launch_fwd<D, DT, true>(a, st)
                                                           : launch_fwd<D, DT, false>(a, st);
}

}  // namespace

int attention_packed_splits(int num_k_tiles, int heads, int kv_heads) {
  const int group = heads / kv_heads;
  const int64_t units = static_cast<int64_t>(num_k_tiles) * kv_heads;
  int splits = 1;
  while (units > 0 && splits < group && units * splits * 2 < 5 * 148) {
    do ++splits; while (group % splits != 0);
  }
  return splits;
}

bool attention_packed_pairs_heads(int heads, int kv_heads) { return (heads / kv_heads) % 2 == 0; }

cudaError_t attention_packed_fwd(const PackedAttnArgs& a, cudaStream_t st) {
  ETHB_TRY(check_common(a), "packed forward");
  ETHB_TRY(check_out(a.o, a.o_strides), "packed forward: out");
  if (a.rows == 0) return cudaSuccess;
  const bool bf = a.dtype == kBF16;
  if (a.head_dim == 128) return bf ? launch_fwd_for<128, kBF16>(a, st) : launch_fwd_for<128, kF16>(a, st);
  return bf ? launch_fwd_for<64, kBF16>(a, st) : launch_fwd_for<64, kF16>(a, st);
}

cudaError_t attention_packed_bwd(const PackedAttnArgs& a, cudaStream_t st) {
  ETHB_TRY(check_common(a), "packed backward");
  ETHB_TRY(check_out(a.o, a.o_strides), "packed backward: out");
  ETHB_RETURN_IF(a.counters == nullptr || a.splits < 1 || (a.heads / a.kv_heads) % a.splits != 0 ||
                     (a.splits > 1 && a.parts == nullptr), cudaErrorInvalidValue, "packed backward: workspace");
  ETHB_TRY(check_out(a.dq, a.dq_strides), "packed backward: dq");
  ETHB_TRY(check_out(a.dk, a.dk_strides), "packed backward: dk");
  ETHB_TRY(check_out(a.dv, a.dv_strides), "packed backward: dv");
  if (a.rows == 0) return cudaSuccess;
  const bool bf = a.dtype == kBF16;
  if (a.head_dim == 128) return bf ? launch_bwd<128, kBF16>(a, st) : launch_bwd<128, kF16>(a, st);
  return bf ? launch_bwd<64, kBF16>(a, st) : launch_bwd<64, kF16>(a, st);
}

}  // namespace ethb
