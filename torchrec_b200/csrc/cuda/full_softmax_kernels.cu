// Cross entropy of a softmax over a whole catalogue, with its gradient, without keeping the scores.  For the rows i whose target is
// not ignored (z = h W^T + b, all sums in fp32, operands bf16):
//   loss_i = log sum_v exp z_iv - z_i,t          dW = G^T h,  db = sum_i G,  dh = G W,   G_iv = g_i (exp(z_iv - lse_i) - [v = t_i]).
// A library route writes the [P, V] scores and reads them back several times; here a 128 x 128 tile of them lives in tensor memory.
//
// One kernel, three forms.  128 rows X stay in shared memory, 128-row tiles Y are streamed past them:
//   S = X Y^T (tcgen05, fp32 in TMEM) -> E = f(S) in registers, rounded to bf16, written back over S -> ACC += E Y (A operand in TMEM).
//   FWD  X = rows of h, Y = W.   f is the running softmax, so that ACC / sum is the expectation of W under the softmax: the forward
//        already holds dh up to the upstream factor, and no pass over the scores is spent on dh in the backward.
//   LSE  the same without ACC (no gradient wanted).
//   BWD  X = rows of W, Y = h.   f uses the known log sum, so ACC = dW of the 128 items; nothing is added up across blocks.
// That is 8 P V D operations for the step, of which 2 P V D recompute the scores, and two exponentials per score.
// The target's own term never enters the rounded sums: with w = 1 - p_t (from the sum over the others), dh = w (ACC / sum - W_t) and
// G_it = -w, so rows that the model already predicts well keep their relative accuracy.
//
// E, and G in the backward, are rounded to bf16 (by at most 2^-8 of a term) in front of the second product, as the first one's operands are:
// the terms need an exponent range that fp16 has not, and a tf32 product would run at half the rate and want W and h in 32 bits too.  The sums
// are of the terms before that rounding, and like ACC in fp32; gradients that leave in fp32 hold the same rounded terms.
//
// Both products want the streamed tile, once K-major (S) and once MN-major (ACC); one copy in shared memory serves both up to
// D = 256, where ACC takes the 256 TMEM columns that two S tiles leave.  Wider rows are cut into pieces of 256 columns that
// recompute S (and load the tile twice).
// The reference of a row's exponentials is raised lazily: ACC and the sums are rescaled only when a row's maximum grew by more than 2^40.
// It is a whole power of two next to zero, and counts from one of the row's own scores where those are far from zero (FsRef): classes masked
// by a large finite bias give no infinities, and a row in which all of them are masked alike is the uniform softmax that it is.
// Ignored rows are left out at the start (their h is never multiplied, so NaN or infinity in padding does not spread) and cost nothing.
// All sums run in a fixed order: pieces of the streamed axis go to a workspace and are joined by a second kernel.
// Every wait is bounded (tcgen05.cuh); a block that gives up raises an error word, marks the call's state and returns, and the kernels behind
// it give NaN for the loss and every gradient of that call.
//
// Measured (B200, 18944 rows x 40000 classes, whole forward or backward): D = 256 forward with dh 657 us (1.18 PFLOP/s), backward 576 us
// (1.35), value only 380 us (1.02); D = 64 448, 328 and 372 us; D = 512 (half the rows) 907, 933 and 277 us, with the scores computed once per
// 256 columns, and D = 1024 (a quarter) 1860, 1803 and 380 us.  At 16384 x 131071 x 256 a step takes 4.27 ms: 8 P V D at 1.03 PFLOP/s under the
// power cap (the library product alone sustains 1.40).  What bounds it: the score product reads both operands from shared memory, which
// also receives the streamed tile.  Narrow rows and values alone take 1.1 to 1.2 us a tile whatever D is; what bounds them is not known: the
// special-function pipe is 47 to 56 % busy, 0.45 instructions are issued a cycle, most stalls are the fixed latency between dependent
// instructions, and more warps, paired arithmetic or a polynomial for a part of the exponentials each left the time as it was.
//
// (The reference ends BERT4Rec in a dense projection over the vocabulary and nn.CrossEntropyLoss, examples/bert4rec/bert4rec_main.py.)
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"
#include "transformer_ops.h"

namespace trb {

constexpr int kFsTile = 128;                        // rows of X, and of a streamed tile
constexpr int kFsThreads = 320;                     // TMA warp, MMA warp, 8 softmax warps
constexpr int kFsSlotBytes = kFsTile * 128;         // 128 rows x 64 bf16
constexpr int kFsSlots = 14;                        // X and the ring of streamed blocks
constexpr int kFsMaxUnits = 13;
constexpr int kFsMaxD = 1024;
constexpr int kFsAcc = 256;                         // accumulator columns
constexpr int kFsExtra = 3 * 1024;                  // per-column values of a tile, exchange of maxima, barriers
constexpr int kFsSmem = kFsSlots * kFsSlotBytes + kFsExtra;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Base-2 growth of a row's maximum that forces a rescale.  The terms have bf16's and fp32's exponents: 2^40 over 2^31 columns is far
// from overflow, and what is flushed lies 2^86 below the largest term.
constexpr float kRaise = 40.f;

// Scores beyond this size are compared with a score of the row before they are scaled to base 2: z log2(e) and its rounding, which the
// reference would be, lie up to 2^-24 |z| apart, for a mask of -1e10 hundreds of powers of two.  Below it the reference is an exact whole number.
constexpr float kFar = 4194304.f;  // 2^22

enum FsMode : int { FS_LSE = 0, FS_FWD = 1, FS_BWD = 2 };
enum FsErr : int { FS_ERR_EMPTY = 1, FS_ERR_FULL = 2, FS_ERR_X = 3, FS_ERR_S = 4, FS_ERR_P = 5, FS_ERR_ACC = 6, FS_ERR_COL = 7, FS_ERR_XCH = 8, FS_ERR_SMEM = 9, FS_ERR_TARGET = 16 };

__device__ int g_fs_error = 0;  // one word per device; never allocated, so it may first be touched inside a graph capture

// The kernels of a call are launched so that the next one may begin (and set itself up) before the one in front has ended; what that one
// wrote is read behind fs_after.  fs_let_next allows the next kernel's blocks in as soon as all of this kernel's have started.
__device__ __forceinline__ void fs_after() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void fs_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename Kernel, typename... Args>
static void fs_launch_next(Kernel kernel, unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  TRB_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
}

// How the work is dealt to the blocks.  An item is a tile of X and a piece of the accumulator's columns; it streams `ty` tiles of Y.  Every
// block takes the same number of whole items, and what is left over (fewer items than blocks) is cut along the streamed axis into one equal
// run per block, which may cross from one item into the next: with whole items alone 313 items keep 148 SMs busy 70 % of the time.
// Blocks work on whole items in step, so that a streamed tile that one of them fetched is in L2 for the others.  Computed alike by every
// kernel (the number of rows that are not ignored is only known on the device), in whole numbers.
struct FsSchedule {
  int tx, ty, steps, whole, rest, run;  // steps: tiles of an item, at least 1; whole: items per block; rest: items left over; run: steps of a block's share of them

  __host__ __device__ FsSchedule(int nx, int ny, int pieces, int grid) {
    tx = (nx + kFsTile - 1) / kFsTile;
    ty = (ny + kFsTile - 1) / kFsTile;
    steps = ty > 0 ? ty : 1;
    whole = tx * pieces / grid;
    rest = tx * pieces - whole * grid;
    run = int((int64_t(rest) * steps + grid - 1) / grid);
  }
  // the runs that an item left over (`rel`: counted from the first of them) is cut into
  __host__ __device__ int first_run(int rel) const { return int(int64_t(rel) * steps / run); }
  __host__ __device__ int last_run(int rel) const { return int((int64_t(rel + 1) * steps - 1) / run); }
};

// A block's share.  Every part of an item has a slot for partial results: whole items their own number, the parts of items left over
// (number of whole items) + rel + run.
struct FsWalk {
  int block, grid, k = 0, item = 0, t0 = 0, nt = 0, slot = 0;
  bool all = false;  // the item is not cut
  int64_t at, end;

  __device__ FsWalk(const FsSchedule& sc, int block_, int grid_) : block(block_), grid(grid_) {
    at = int64_t(block) * sc.run;
    end = min(at + sc.run, int64_t(sc.rest) * sc.steps);
  }
  __device__ bool next(const FsSchedule& sc) {
    if (k < sc.whole) {
      item = slot = k * grid + block;
      ++k;
      t0 = 0;
      nt = sc.ty;
      all = true;
      return true;
    }
    if (at >= end) return false;
    const int rel = int(at / sc.steps);
    t0 = int(at - int64_t(rel) * sc.steps);
    nt = int(min(int64_t(sc.steps - t0), end - at));
    at += nt;
    item = sc.whole * grid + rel;
    slot = item + block;
    all = nt == sc.steps;
    nt = min(nt, sc.ty);  // no tiles at all: an item without terms
    return true;
  }
};

struct FsParams {
  const int* n_valid;      // rows of h that take part
  int V, D;
  int kb;                  // blocks of 64 columns
  int x_resident, hold;    // X stays in shared memory; a streamed tile stays until ACC has read it
  int grid;
  const int* target;       // [Ppad] targets of the compacted rows
  const float* bias;       // [Vpad] (-inf behind V), or null
  float* part_acc;         // [slots, 128, min(D, 256)]; BWD: of the items left over only
  float2* part_m;          // [slots, 2, 128]  reference (k, base) of either group of warps
  float* part_l;           // [slots, 2, 128]  their sums; BWD: db
  float* zt;               // [Ppad] score of the target
  const float* lse2;       // BWD [Ppad] log sum less its base, base 2 (+inf behind n_valid)
  const float* lbase;      // BWD [Ppad] base of the log sum
  const int* far;          // BWD: not 0 when some row's base is not
  int* gave_up;            // set by a block that gave up
  const float* wex;        // BWD [Ppad] 1 - p_t
  const float* gcol;       // BWD [Ppad] upstream gradient of every row, or null
  const float* dloss;      // BWD scalar upstream gradient (with gcol: unused)
  int mean;                // BWD: divide by n_valid
  void* dw;                // BWD [V, D]
  int dw_fp32;
};

__device__ __forceinline__ float fs_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's reference: a term is 2^((z - base) log2(e) - k).  k is a whole number and base 0 unless the row's scores lie beyond kFar, so that
// rescaling by the difference of two references is exact.  (Beyond it the scores themselves are a quarter and more apart.)
struct FsRef {
  float k = -INFINITY, base = 0.f;
  __device__ __forceinline__ bool is(const FsRef& o) const { return k == o.k && base == o.base; }
  // the largest score that may stand under it
  __device__ __forceinline__ float limit() const { return fmaf(k + kRaise, kLn2, base); }
};
__device__ __forceinline__ float fs_gap(const FsRef& a, const FsRef& b) { return fmaf(a.base - b.base, kLog2e, a.k - b.k); }
// what terms under `from` are multiplied by to stand under `to`
__device__ __forceinline__ float fs_factor(const FsRef& from, const FsRef& to) { return from.is(to) ? 1.f : fs_ex2(fs_gap(from, to)); }
// the same in either order
__device__ __forceinline__ FsRef fs_higher(const FsRef& a, const FsRef& b) {
  const float g = fs_gap(a, b);
  return g > 0.f || (g == 0.f && a.base > b.base) ? a : b;
}
// the reference at `top`, a score above the old one
__device__ __forceinline__ FsRef fs_raised(const FsRef& r, float top) {
  FsRef n;
  if (fabsf(top) < kFar) {
    n.k = ceilf(top * kLog2e);
  } else if (r.base != 0.f && fabsf(top - r.base) < kFar) {
    n.base = r.base;
    n.k = ceilf((top - r.base) * kLog2e);
  } else {
    n.base = top;
    n.k = 0.f;
  }
  return n;
}

__device__ __forceinline__ uint32_t fs_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void fs_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}

__host__ __device__ constexpr uint32_t fs_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(kFsTile >> 4) << 24);
}

struct FsBars {
  uint64_t full[kFsMaxUnits], empty[kFsMaxUnits];
  uint64_t x_full, x_empty;
  uint64_t s_full[4], p_full[4];
  uint64_t acc_done[4], o_empty;  // acc_done by the tile's number: a waiter may know no more than that the product four tiles back is done
  uint64_t c_full[4], c_empty[4];
  uint64_t m_done[4], drain;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(FsBars) + 2048 <= kFsExtra, "the shared memory behind the slots is too small");

// The part of a wait that loops is kept out of line: the roles' loops have to stay within the instruction caches.
__device__ __noinline__ bool fs_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  return mbar_wait(bar, parity, abort_flag, &g_fs_error, code);
}
__device__ __forceinline__ bool fs_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  return mbar_try_wait(bar, parity) || fs_wait_long(bar, parity, abort_flag, code);
}

// position in the ring of streamed blocks
struct FsRing {
  uint32_t units, stage = 0, phase = 0;
  __device__ explicit FsRing(uint32_t n) : units(n) {}
  __device__ void next() {
    if (++stage == units) {
      stage = 0;
      phase ^= 1;
    }
  }
};

template <int MODE, bool BIAS, bool ROWG>
__global__ void __launch_bounds__(kFsThreads, 1)
full_softmax_kernel(const __grid_constant__ CUtensorMap tmapX, const __grid_constant__ CUtensorMap tmapY, const FsParams p) {
  constexpr bool kAcc = MODE != FS_LSE;
  constexpr uint32_t kTmemCols = 512;
  // Score tiles in TMEM: two beside an accumulator of up to 256 columns, three beside one of up to 128 (S then runs two tiles ahead, so
  // that neither group of softmax warps waits for the products of the tile that it has just handed over: rows of 64 to 128 values are
  // bound by the exponentials), four without an accumulator.
  const uint32_t bufs = kAcc ? (p.D <= 128 ? 3 : 2) : 4;
  const uint32_t o_col = bufs * kFsTile;
  constexpr uint32_t kCols = ROWG ? 2 : 4, kColShift = ROWG ? 1 : 2;  // tiles whose per-column values are in shared memory
  constexpr int kPair = kAcc ? 1 : 2;  // without an accumulator two tiles are one product of 256 columns, which reads X half as often
  extern __shared__ __align__(1024) uint8_t fs_smem[];
  float* cols = reinterpret_cast<float*>(fs_smem + kFsSlots * kFsSlotBytes);  // FWD: the rows' references, k [128], base [128]; BWD: lse2 [4][128], or lse2 [2][128], g [2][128]
  FsBars* B = reinterpret_cast<FsBars*>(cols + 512);
  volatile int* abort_flag = &B->abort_flag;
  // values that are alike in a warp are taken from lane 0, which tells the compiler so
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  // a unit of the ring: two blocks of 64 columns of a tile (one for rows of up to 64), or one block of a pair of tiles
  const int spu = kAcc && p.kb == 1 ? 1 : 2;               // its slots
  const int upt = kAcc ? (p.kb + spu - 1) / spu : p.kb;    // units of a streamed tile or pair
  const int x_slots = p.x_resident ? p.kb : 0;
  const uint32_t units = min((kFsSlots - x_slots) / spu, kFsMaxUnits);
  uint8_t* ring = fs_smem + x_slots * kFsSlotBytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kFsMaxUnits; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->empty[i], 1);
    }
    mbar_init(&B->x_full, 1);
    mbar_init(&B->x_empty, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&B->s_full[i], 1);
      mbar_init(&B->p_full[i], 4);
      mbar_init(&B->m_done[i], 1);
      mbar_init(&B->acc_done[i], 1);
      mbar_init(&B->c_full[i], 1);
      mbar_init(&B->c_empty[i], 4);
    }
    mbar_init(&B->o_empty, 8);
    mbar_init(&B->drain, 1);
    *abort_flag = 0;
    // the swizzled descriptors want slots on 1024-byte boundaries
    if ((smem_u32(fs_smem) & 1023) != 0) {
      *abort_flag = 1;
      atomicCAS(&g_fs_error, 0, FS_ERR_SMEM);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B->tmem_base)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  fs_after();
  const int n_valid = __shfl_sync(0xffffffffu, *p.n_valid, 0);
  const int nx = MODE == FS_BWD ? p.V : n_valid, ny = MODE == FS_BWD ? n_valid : p.V;
  const FsSchedule sc(nx, ny, kAcc ? (p.D + kFsAcc - 1) / kFsAcc : 1, p.grid);
  const uint32_t tmem = __shfl_sync(0xffffffffu, B->tmem_base, 0);
  bool ok = *abort_flag == 0;

  FsWalk walk(sc, blockIdx.x, p.grid);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      FsRing r(units);
      uint32_t item = 0, tc = 0, loads = 0;
      auto load_unit = [&](const CUtensorMap* map, int u, int row, bool pair) {
        if (!fs_wait(&B->empty[r.stage], r.phase ^ 1, abort_flag, FS_ERR_EMPTY)) return false;
        const int n = kAcc ? min(spu, p.kb - u * spu) : (pair ? 2 : 1), col = kAcc ? u * spu * 64 : u * 64;
        uint8_t* dst = ring + r.stage * spu * kFsSlotBytes;
        mbar_expect_tx(&B->full[r.stage], n * kFsSlotBytes);
        tma_load_2d(dst, map, &B->full[r.stage], col, row);
        if (n > 1) tma_load_2d(dst + kFsSlotBytes, map, &B->full[r.stage], kAcc ? col + 64 : col, kAcc ? row : row + kFsTile);
        r.next();
        ++loads;
        return true;
      };
      for (; ok && walk.next(sc); ++item) {
        const int x = walk.item % sc.tx, piece = walk.item / sc.tx, t0 = walk.t0, nt = walk.nt;
        if (p.x_resident && nt > 0) {
          if (item > 0 && !fs_wait(&B->x_empty, (item - 1) & 1, abort_flag, FS_ERR_X)) { ok = false; break; }
          mbar_expect_tx(&B->x_full, p.kb * kFsSlotBytes);
          for (int k = 0; k < p.kb; ++k) tma_load_2d(fs_smem + k * kFsSlotBytes, &tmapX, &B->x_full, k * 64, x * kFsTile);
        }
        const int pu0 = piece * (kFsAcc / 128), pu1 = min(upt, pu0 + kFsAcc / 128);
        const int groups = (nt + kPair - 1) / kPair, ahead = kAcc ? int(bufs) - 1 : 0;
        for (int t = 0; t < groups + ahead && ok; ++t) {
          if (t < groups) {
            for (int u = 0; u < upt && ok; ++u) {
              if (!p.x_resident) ok = load_unit(&tmapX, u, x * kFsTile, false);
              ok = ok && load_unit(&tmapY, u, (t0 + t * kPair) * kFsTile, true);  // behind the last row zeros arrive
            }
            if constexpr (MODE == FS_BWD) {  // after the tile, whose product does not need them
              const uint32_t b = tc & (kCols - 1);
              if (!ok || !fs_wait(&B->c_empty[b], ((tc >> kColShift) & 1) ^ 1, abort_flag, FS_ERR_COL)) { ok = false; break; }
              mbar_expect_tx(&B->c_full[b], ROWG ? 1024 : 512);
              fs_bulk_load(cols + b * 128, p.lse2 + int64_t(t0 + t) * kFsTile, 512, &B->c_full[b]);
              if constexpr (ROWG) fs_bulk_load(cols + 256 + b * 128, p.gcol + int64_t(t0 + t) * kFsTile, 512, &B->c_full[b]);
              ++tc;
            }
          }
          if (kAcc && !p.hold && t >= ahead)
            for (int u = pu0; u < pu1 && ok; ++u) ok = load_unit(&tmapY, u, (t0 + t - ahead) * kFsTile, true);
        }
      }
      if (!ok) {
        // copies may still be on their way into shared memory: give them a bounded time to land before the block may exit
        const long long begin = clock64();
        for (uint32_t j = loads > units ? loads - units : 0; j < loads; ++j)
          while (!mbar_try_wait(&B->full[j % units], (j / units) & 1) && clock64() - begin < kWaitCycles) {
          }
        if (p.x_resident)
          while (!mbar_try_wait(&B->x_full, item & 1) && clock64() - begin < kWaitCycles) {
          }
        if constexpr (MODE == FS_BWD)
          for (uint32_t j = tc > kCols ? tc - kCols : 0; j < tc; ++j)
            while (!mbar_try_wait(&B->c_full[j & (kCols - 1)], (j >> kColShift) & 1) && clock64() - begin < kWaitCycles) {
            }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // S of the next one or two tiles is issued before ACC(t), so the tensor cores work while the softmax warps turn S(t) into E(t).  Descriptors advance by
    // additions (addresses in units of 16 bytes).  The whole warp runs the loop, one elected lane issues.
    {
      const uint32_t leader = elect_one();
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, fs_wait(bar, parity, abort_flag, code)) != 0;
      };
      FsRing r(units);
      uint32_t item = 0, tc = 0;  // tc: tile whose E is multiplied next
      constexpr uint32_t idesc_s = fs_idesc(kPair * kFsTile, false);
      uint32_t sb = 0, sb_use = 0, eb = 0, eb_phase = 0;  // buffer of the next S and how often it was used, buffer and phase of the next E
      constexpr uint32_t kSlot16 = kFsSlotBytes / 16;
      const uint64_t desc_k = make_smem_desc(0, 16, 1024), desc_mn = make_smem_desc(0, kFsSlotBytes, 1024);
      const uint32_t x16 = smem_u32(fs_smem) >> 4, ring16 = smem_u32(ring) >> 4, unit16 = spu * kSlot16;
      // 64 columns as four products of 16 (the last of them may hold zero columns only)
      auto score_block = [&](uint32_t d, uint64_t dx, uint64_t dy, bool first) {
#pragma unroll
        for (int i = 0; i < 4; ++i) umma_bf16_by(leader, d, dx + i * 2, dy + i * 2, idesc_s, (i > 0 || !first) ? 1u : 0u);
      };
      // rows of up to 256: what does not change from tile to tile
      const uint32_t n0 = min(64 * spu, (p.D + 15) / 16 * 16), n_all = (p.D + 15) / 16 * 16;
      const uint32_t idesc_0 = fs_idesc(n0, true), idesc_1 = fs_idesc(n_all > 128 ? n_all - 128 : 16, true), idesc_all = fs_idesc(n_all & 0x1ff, true);
      const bool two_units = upt == 2, slot_1 = p.kb > 1, slot_3 = p.kb > 3;
      for (; ok && walk.next(sc); ++item) {
        const int piece = walk.item / sc.tx, nt = walk.nt;
        if (p.x_resident && nt > 0 && !wait_all(&B->x_full, item & 1, FS_ERR_X)) { ok = false; break; }
        const int pu0 = piece * (kFsAcc / 128), pu1 = min(upt, pu0 + kFsAcc / 128);
        const int groups = (nt + kPair - 1) / kPair, ahead = kAcc ? int(bufs) - 1 : 0;
        uint32_t held = r.stage;  // first unit of the tile whose E is multiplied next
        if (kAcc && p.hold) {
          for (int t = 0; t < groups + ahead; ++t) {
            if (t < groups) {
              const uint32_t d = tmem + sb * kFsTile;
              if (!wait_all(&B->full[r.stage], r.phase, FS_ERR_FULL)) { ok = false; break; }
              uint64_t dy = desc_k + ring16 + r.stage * unit16;
              r.next();
              score_block(d, desc_k + x16, dy, true);
              if (slot_1) score_block(d, desc_k + x16 + kSlot16, dy + kSlot16, false);
              if (two_units) {
                if (!wait_all(&B->full[r.stage], r.phase, FS_ERR_FULL)) { ok = false; break; }
                dy = desc_k + ring16 + r.stage * unit16;
                r.next();
                score_block(d, desc_k + x16 + 2 * kSlot16, dy, false);
                if (slot_3) score_block(d, desc_k + x16 + 3 * kSlot16, dy + kSlot16, false);
              }
              tcgen05_commit_by(leader, &B->s_full[sb]);
              if (t == groups - 1) tcgen05_commit_by(leader, &B->x_empty);
              if (++sb == bufs) sb = 0;
            }
            if (t >= ahead) {
              const uint32_t more = t == ahead ? 0u : 1u;
              if (more == 0 && item > 0 && !wait_all(&B->o_empty, (item - 1) & 1, FS_ERR_ACC)) { ok = false; break; }
              if (!wait_all(&B->p_full[eb], eb_phase, FS_ERR_P)) { ok = false; break; }
              tcgen05_fence_after();
              const uint32_t e = tmem + eb * kFsTile;
              const uint32_t next = held + 1 == units ? 0 : held + 1;
              const uint64_t dy = desc_mn + ring16 + held * unit16;
              if (two_units && next != 0) {  // both units of the tile in one product where they lie side by side in the ring
#pragma unroll
                for (int i = 0; i < 8; ++i) umma_bf16_ts_by(leader, tmem + o_col, e + i * 8, dy + i * 128, idesc_all, i > 0 ? 1u : more);
                tcgen05_commit_by(leader, &B->empty[held]);
                tcgen05_commit_by(leader, &B->empty[next]);
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) umma_bf16_ts_by(leader, tmem + o_col, e + i * 8, dy + i * 128, idesc_0, i > 0 ? 1u : more);
                tcgen05_commit_by(leader, &B->empty[held]);
                if (two_units) {
                  const uint64_t dy1 = desc_mn + ring16 + next * unit16;
#pragma unroll
                  for (int i = 0; i < 8; ++i) umma_bf16_ts_by(leader, tmem + o_col + 128, e + i * 8, dy1 + i * 128, idesc_1, i > 0 ? 1u : more);
                  tcgen05_commit_by(leader, &B->empty[next]);
                }
              }
              held = two_units ? (next + 1 == units ? 0 : next + 1) : next;
              tcgen05_commit_by(leader, &B->acc_done[tc & 3]);
              ++tc;
              if (++eb == bufs) {
                eb = 0;
                eb_phase ^= 1;
              }
            }
          }
          continue;
        }
        // wider rows, or no accumulator: blocks are given back as soon as they were multiplied, and loaded again for the accumulator
        const uint32_t n_first = min(128, (p.D - pu0 * 128 + 15) / 16 * 16), n_second = min(128, (p.D - pu0 * 128 - 128 + 15) / 16 * 16);
        const uint32_t idesc_first = fs_idesc(n_first, true), idesc_second = fs_idesc(n_second, true);
        const bool second = pu1 - pu0 == 2;
        for (int t = 0; t < groups + ahead; ++t) {
          if (t < groups) {
            // the buffer's previous tile: with ACC its E was consumed by an MMA issued before this one; without, its readers must be done
            if constexpr (!kAcc) {
              if (sb_use > 0 && (!wait_all(&B->p_full[sb], (sb_use - 1) & 1, FS_ERR_P) || !wait_all(&B->p_full[sb + 1], (sb_use - 1) & 1, FS_ERR_P))) { ok = false; break; }
              tcgen05_fence_after();
            }
            const uint32_t d = tmem + sb * kFsTile;
            uint64_t dx = desc_k + x16;
            for (int u = 0; u < upt; ++u) {
              const uint32_t xs = r.stage;
              if (!p.x_resident) {
                if (!wait_all(&B->full[xs], r.phase, FS_ERR_FULL)) { ok = false; break; }
                dx = desc_k + ring16 + xs * unit16;
                r.next();
              }
              const uint32_t ys = r.stage;
              if (!wait_all(&B->full[ys], r.phase, FS_ERR_FULL)) { ok = false; break; }
              r.next();
              const uint64_t dy = desc_k + ring16 + ys * unit16;
              score_block(d, dx, dy, u == 0);
              if (kAcc && 2 * u + 1 < p.kb) score_block(d, dx + kSlot16, dy + kSlot16, false);
              if (!p.x_resident) tcgen05_commit_by(leader, &B->empty[xs]);
              tcgen05_commit_by(leader, &B->empty[ys]);
              dx += kAcc ? unit16 : kSlot16;
            }
            if (!ok) break;
            tcgen05_commit_by(leader, &B->s_full[sb]);
            if constexpr (!kAcc) tcgen05_commit_by(leader, &B->s_full[sb + 1]);
            if (p.x_resident && t == groups - 1) tcgen05_commit_by(leader, &B->x_empty);
            sb += kPair;
            if (sb == bufs) {
              sb = 0;
              ++sb_use;
            }
          }
          if (kAcc && t >= ahead) {
            const uint32_t more = t == ahead ? 0u : 1u;
            if (more == 0 && item > 0 && !wait_all(&B->o_empty, (item - 1) & 1, FS_ERR_ACC)) { ok = false; break; }
            if (!wait_all(&B->p_full[eb], eb_phase, FS_ERR_P)) { ok = false; break; }
            tcgen05_fence_after();
            const uint32_t e = tmem + eb * kFsTile;
            if (!wait_all(&B->full[r.stage], r.phase, FS_ERR_FULL)) { ok = false; break; }
            uint64_t dy = desc_mn + ring16 + r.stage * unit16;
#pragma unroll
            for (int i = 0; i < 8; ++i) umma_bf16_ts_by(leader, tmem + o_col, e + i * 8, dy + i * 128, idesc_first, i > 0 ? 1u : more);
            tcgen05_commit_by(leader, &B->empty[r.stage]);
            r.next();
            if (second) {
              if (!wait_all(&B->full[r.stage], r.phase, FS_ERR_FULL)) { ok = false; break; }
              dy = desc_mn + ring16 + r.stage * unit16;
#pragma unroll
              for (int i = 0; i < 8; ++i) umma_bf16_ts_by(leader, tmem + o_col + 128, e + i * 8, dy + i * 128, idesc_second, i > 0 ? 1u : more);
              tcgen05_commit_by(leader, &B->empty[r.stage]);
              r.next();
            }
            tcgen05_commit_by(leader, &B->acc_done[tc & 3]);
            ++tc;
            if (++eb == bufs) {
              eb = 0;
              eb_phase ^= 1;
            }
          }
        }
      }
      if (!ok) {  // products already issued must end before the tensor memory is freed
        tcgen05_commit_by(leader, &B->drain);
        const long long begin = clock64();
        while (!mbar_try_wait(&B->drain, 0) && clock64() - begin < kWaitCycles) {
        }
      }
    }
  } else {
    // ---------------- softmax warps (2..9) ----------------
    // Two groups of four warps take the tiles in turn (group = parity of the tile), so that one group's exponentials fill the other's
    // waits; a thread owns a row of the tile (TMEM lane quarter = warp % 4) and walks its 128 columns in pieces of 32.  The loop over
    // the pieces is not unrolled: with the tile unrolled the warps waited for instructions a third of the time.
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    uint32_t item = 0, tc = 0;
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, fs_wait(bar, parity, abort_flag, code)) != 0;
    };
    for (; ok && walk.next(sc); ++item) {
      const int x = walk.item % sc.tx, piece = walk.item / sc.tx, t0 = walk.t0, nt = walk.nt;
      const int row = x * kFsTile + q * 32 + lane;  // FWD: compacted row of h; BWD: item
      const int r128 = q * 32 + lane;
      int tgt = -1;
      float bias_row = 0.f;
      const bool far = MODE == FS_BWD && __shfl_sync(0xffffffffu, *p.far, 0) != 0;
      if constexpr (MODE == FS_BWD) {
        if constexpr (BIAS) bias_row = far ? 0.f : p.bias[row] * kLog2e;  // padded to whole tiles
      } else {
        tgt = p.target[row];
      }
      FsRef ref;
      float l = 0.f, limit = -INFINITY;
      const uint32_t tc0 = tc, tc1 = tc + (nt + kPair - 1) / kPair * kPair;
      tc += (tc ^ half) & 1;
      uint32_t b = tc % bufs, ph = (tc / bufs) & 1;  // the tile's buffer
      auto next_buffer = [&] {
        b += 2;
        if (b >= bufs) {
          b -= bufs;
          ph ^= 1;
        }
      };
      for (; tc < tc1 && ok; tc += 2, next_buffer()) {
        const int t = int(tc - tc0);
        const int col0 = (t0 + t) * kFsTile;
        if (!wait_all(&B->s_full[b], ph, FS_ERR_S)) { ok = false; break; }
        tcgen05_fence_after();
        if (!kAcc && t >= nt) {  // the pair's second tile lies behind the last
          if (lane == 0) mbar_arrive(&B->p_full[b]);
          continue;
        }
        const uint32_t ts = tmem + lanes + b * kFsTile;
        uint32_t r[32];
        tmem_ld_32x32_issue(ts, r);
        if constexpr (MODE == FS_BWD) {
          const int v0 = x * kFsTile + q * 32;
          int tg = p.target[col0 + lane];  // targets of 32 rows of h, one per lane
          const uint32_t cb = tc & (kCols - 1);
          if (!wait_all(&B->c_full[cb], (tc >> kColShift) & 1, FS_ERR_COL)) { ok = false; break; }
          auto tile = [&](auto far_rows) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float z[32];
              tmem_ld_wait(r);
              const float4* lp = reinterpret_cast<const float4*>(cols + cb * 128 + c * 32);
              if constexpr (decltype(far_rows)::value) {  // scores less the base of their row's log sum
                const float4* fp = reinterpret_cast<const float4*>(p.lbase + col0 + c * 32);
                const float bias_far = BIAS ? p.bias[row] : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 v = fp[j];
                  r[4 * j] = __float_as_uint(__uint_as_float(r[4 * j]) + bias_far - v.x);
                  r[4 * j + 1] = __float_as_uint(__uint_as_float(r[4 * j + 1]) + bias_far - v.y);
                  r[4 * j + 2] = __float_as_uint(__uint_as_float(r[4 * j + 2]) + bias_far - v.z);
                  r[4 * j + 3] = __float_as_uint(__uint_as_float(r[4 * j + 3]) + bias_far - v.w);
                }
              }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 v = lp[j];
                const float s4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float s = __uint_as_float(r[4 * j + k]);
                  z[4 * j + k] = BIAS ? fmaf(s, kLog2e, bias_row) - s4[k] : fmaf(s, kLog2e, -s4[k]);
                }
              }
              // entries (item, row of h) with the row's target: p - 1 = -(1 - p_t)
              uint32_t hits = __ballot_sync(0xffffffffu, tg >= v0 && tg < v0 + 32);
              const int tg_now = tg;
              if (c < 3) {
                tmem_ld_32x32_issue(ts + (c + 1) * 32, r);
                tg = p.target[col0 + (c + 1) * 32 + lane];
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) z[j] = fs_ex2(z[j]);
              while (hits) {
                const int j = __ffs(hits) - 1;
                hits &= hits - 1;
                if (__shfl_sync(0xffffffffu, tg_now, j) == v0 + lane) {
                  const float v = -p.wex[col0 + c * 32 + j];
#pragma unroll
                  for (int k = 0; k < 32; ++k) z[k] = k == j ? v : z[k];
                }
                __syncwarp();
              }
              if constexpr (ROWG) {
                const float4* gp = reinterpret_cast<const float4*>(cols + 256 + cb * 128 + c * 32);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 v = gp[j];
                  z[4 * j] *= v.x;
                  z[4 * j + 1] *= v.y;
                  z[4 * j + 2] *= v.z;
                  z[4 * j + 3] *= v.w;
                }
              }
              if constexpr (BIAS) {
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[j & 3] += z[j];
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
              }
              // E of these columns over score columns that this thread has read already
              uint32_t e[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) e[j] = fs_pack(z[2 * j], z[2 * j + 1]);
              tmem_st_32x16(ts + c * 16, e);
            }
          };
          // (with the rare case inside the loop of the other one: 324 -> 363 us, 18944 x 40000 x 64 with a bias)
          if (far) tile(std::true_type());
          else tile(std::false_type());
          __syncwarp();
          if (lane == 0) mbar_arrive(&B->c_empty[cb]);
        } else {
          const int rel = tgt - col0;  // the target's column in this tile
          const bool any_hit = __any_sync(0xffffffffu, tgt >= 0 && rel >= 0 && rel < kFsTile);
          // multiplies the terms of this tile that are stored already
          auto rescale_terms = [&](int pieces, float f) {
            tmem_st_wait();
#pragma unroll 1
            for (int k = 0; k < pieces; ++k) {
              uint32_t a[16];
              tmem_ld_32x16_issue(ts + k * 16, a);
              tmem_ld_wait(a);
#pragma unroll
              for (int j = 0; j < 16; ++j) a[j] = fs_pack(__uint_as_float(a[j] << 16) * f, __uint_as_float(a[j] & 0xffff0000u) * f);
              tmem_st_32x16(ts + k * 16, a);
              tmem_st_wait();
            }
          };
          if constexpr (MODE == FS_FWD) {
            if (t == 1) {  // this group's first tile: the row's reference comes from the tile before
              if (!wait_all(&B->m_done[q], (tc - 1) & 1, FS_ERR_XCH)) { ok = false; break; }
              ref.k = cols[r128];
              ref.base = cols[128 + r128];
              limit = ref.base != 0.f ? -INFINITY : ref.limit();
            }
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float z[32];
            tmem_ld_wait(r);
#pragma unroll
            for (int j = 0; j < 32; ++j) z[j] = __uint_as_float(r[j]);
            if constexpr (BIAS) {
              const float4* bp = reinterpret_cast<const float4*>(p.bias + col0 + c * 32);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 v = bp[j];  // (written by the kernel in front, during this one's life: not through the read-only path)
                z[4 * j] += v.x;
                z[4 * j + 1] += v.y;
                z[4 * j + 2] += v.z;
                z[4 * j + 3] += v.w;
              }
            } else if (__builtin_expect(col0 + kFsTile > p.V, 0)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col0 + c * 32 + j >= p.V) z[j] = -INFINITY;
            }
            if (__builtin_expect(any_hit, 0)) {  // the target's own term stays out
              float zt = 0.f;
              const int at = rel - c * 32;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                zt = j == at ? z[j] : zt;
                z[j] = j == at ? -INFINITY : z[j];
              }
              if (piece == 0 && tgt >= 0 && at >= 0 && at < 32) p.zt[row] = zt;
              __syncwarp();
            }
            float mx[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
            for (int j = 4; j < 32; ++j) mx[j & 3] = fmaxf(mx[j & 3], z[j]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if (__builtin_expect(__any_sync(0xffffffffu, top > limit), 0)) {  // rows whose base is not 0 always come here
              const bool raise = top > ref.limit();
              if (__any_sync(0xffffffffu, raise)) {
                const FsRef now = raise ? fs_raised(ref, top) : ref;
                const float f = fs_factor(ref, now);
                ref = now;
                limit = ref.base != 0.f ? -INFINITY : ref.limit();
                l *= f;
                if constexpr (kAcc) rescale_terms(c, f);
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) z[j] -= ref.base;
            }
            const float ms = ref.k == -INFINITY ? 0.f : ref.k;
#pragma unroll
            for (int j = 0; j < 32; ++j) z[j] = fmaf(z[j], kLog2e, -ms);
            if (c < 3) tmem_ld_32x32_issue(ts + (c + 1) * 32, r);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              z[j] = fs_ex2(z[j]);
              sum[j & 3] += z[j];
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (kAcc) {
              // the terms in bf16 over score columns that this thread has read already
              uint32_t e[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) e[j] = fs_pack(z[2 * j], z[2 * j + 1]);
              tmem_st_32x16(ts + c * 16, e);
            }
          }
          if constexpr (MODE == FS_FWD) {
            // The accumulator and both groups' sums refer to one maximum per row, kept in shared memory: a tile is published after the
            // tile before it, by when that one's decision is known.
            if (t == 0) {
              cols[r128] = ref.k;
              cols[128 + r128] = ref.base;
            } else {
              if (t > 1 && !wait_all(&B->m_done[q], (tc - 1) & 1, FS_ERR_XCH)) { ok = false; break; }
              FsRef acc_ref;
              acc_ref.k = cols[r128];
              acc_ref.base = cols[128 + r128];
              if (__builtin_expect(__any_sync(0xffffffffu, !acc_ref.is(ref)), 0)) {
                const FsRef now = fs_higher(acc_ref, ref);
                const float fe = fs_factor(ref, now);
                l *= fe;
                rescale_terms(4, fe);
                if (__any_sync(0xffffffffu, !now.is(acc_ref))) {
                  // every ACC up to the previous tile has to be complete; this tile's has not been issued
                  if (!wait_all(&B->acc_done[(tc - 1) & 3], ((tc - 1) >> 2) & 1, FS_ERR_ACC)) { ok = false; break; }
                  tcgen05_fence_after();
                  const float f = fs_factor(acc_ref, now);
                  const int groups = (min(kFsAcc, p.D - piece * kFsAcc) + 15) / 16;
#pragma unroll 1
                  for (int g = 0; g < groups; ++g) {
                    const uint32_t to = tmem + lanes + o_col + g * 16;
                    uint32_t a[16];
                    tmem_ld_32x16_issue(to, a);
                    tmem_ld_wait(a);
#pragma unroll
                    for (int j = 0; j < 16; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * f);
                    tmem_st_32x16(to, a);
                  }
                  cols[r128] = now.k;
                  cols[128 + r128] = now.base;
                }
                ref = now;
                limit = ref.base != 0.f ? -INFINITY : ref.limit();
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&B->m_done[q]);
          }
        }
        if constexpr (kAcc) tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->p_full[b]);
      }
      if (!ok) break;
      tc = tc1;
      // ---- end of the item ----
      if constexpr (MODE == FS_FWD) {
        if (nt > 0 && ((tc - 1) & 1) != uint32_t(half)) {  // the other group had the last tile
          if (!wait_all(&B->m_done[q], (tc - 1) & 1, FS_ERR_XCH)) { ok = false; break; }
          FsRef acc_ref;
          acc_ref.k = cols[r128];
          acc_ref.base = cols[128 + r128];
          l *= fs_factor(ref, acc_ref);
          ref = acc_ref;
        }
      }
      if (MODE != FS_BWD || (BIAS && piece == 0)) {
        const int64_t at = (int64_t(walk.slot) * 2 + half) * kFsTile + r128;
        p.part_l[at] = l;
        if constexpr (MODE != FS_BWD) p.part_m[at] = make_float2(ref.k, ref.base);
      }
      if constexpr (kAcc) {
        if (nt > 0) {
          if (!wait_all(&B->acc_done[(tc - 1) & 3], ((tc - 1) >> 2) & 1, FS_ERR_ACC)) { ok = false; break; }
          tcgen05_fence_after();
        }
        const int width = min(kFsAcc, p.D - piece * kFsAcc);
        const bool direct = MODE == FS_BWD && walk.all;
        const int acc_width = min(p.D, kFsAcc);
        float* part = direct ? nullptr : p.part_acc + (int64_t(MODE == FS_BWD ? walk.slot - sc.whole * p.grid : walk.slot) * kFsTile + r128) * acc_width;
        float scale = 1.f;
        if (direct && !ROWG) scale = *p.dloss / (p.mean ? float(max(n_valid, 1)) : 1.f);
        for (int g = half; g * 32 < width; g += 2) {
          uint32_t a[32];
          if (nt > 0) {
            tmem_ld_32x32_issue(tmem + lanes + o_col + g * 32, a);
            tmem_ld_wait(a);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j] = 0u;
          }
          const int c0 = piece * kFsAcc + g * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            if (row >= nx || c0 + j >= p.D) continue;  // D % 8 == 0
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(a[j + k]) * scale;
            if (!direct || p.dw_fp32) {
              float* o = direct ? reinterpret_cast<float*>(p.dw) + int64_t(row) * p.D + c0 + j : part + g * 32 + j;
              *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
              uint4 o = make_uint4(fs_pack(v[0], v[1]), fs_pack(v[2], v[3]), fs_pack(v[4], v[5]), fs_pack(v[6], v[7]));
              *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.dw) + int64_t(row) * p.D + c0 + j) = o;
            }
          }
          __syncwarp();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->o_empty);
      }
    }
    if (!ok) {  // reads and writes of tensor memory on their way must end before it is freed
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      tmem_st_wait();
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag != 0) *p.gave_up = 1;
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---- workspace ----------------------------------------------------------------------------------------
// What the forward leaves for the backward, in one allocation: counters, targets, the rows' places, statistics, the padded bias, the
// compacted rows of h and (with a gradient of h wanted) dh without the upstream factor.
enum FsCounter : int { FS_N_VALID = 0, FS_N_BAD = 1, FS_JOINED = 2, FS_FAR = 3, FS_GAVE_UP = 4, FS_COUNTERS = 8 };

struct FsState {
  int* counters;        // [FS_COUNTERS + Ppad / 128]: joined rows of every tile behind the first ones
  int* target;          // [Ppad] of the compacted rows, -1 behind the last
  int* orig;            // [Ppad] their rows of h
  int* slot;            // [P] place of every row of h, or -1
  float* lse2;          // [Ppad] log sum less its base (base 2), +inf behind the last
  float* lbase;         // [Ppad] base of the log sum, in the scores' units
  float* wex;           // [Ppad] 1 - p_t
  float* bias;          // [Vpad], or null
  __nv_bfloat16* hc;    // [Ppad, Dp]
  float* unit;          // [Ppad, Dp], or null
  int64_t bytes;

  FsState(void* base, int64_t P, int64_t V, int64_t Dp, bool has_bias, bool has_unit) {
    const int64_t Ppad = (P + kFsTile - 1) / kFsTile * kFsTile, Vpad = (V + kFsTile - 1) / kFsTile * kFsTile;
    int64_t at = 0;
    auto take = [&](int64_t n) {
      uint8_t* r = reinterpret_cast<uint8_t*>(base) + at;
      at += (n + 255) / 256 * 256;
      return r;
    };
    counters = reinterpret_cast<int*>(take(4 * (FS_COUNTERS + Ppad / kFsTile)));
    target = reinterpret_cast<int*>(take(4 * Ppad));
    orig = reinterpret_cast<int*>(take(4 * Ppad));
    slot = reinterpret_cast<int*>(take(4 * P));
    lse2 = reinterpret_cast<float*>(take(4 * Ppad));
    lbase = reinterpret_cast<float*>(take(4 * Ppad));
    wex = reinterpret_cast<float*>(take(4 * Ppad));
    bias = has_bias ? reinterpret_cast<float*>(take(4 * Vpad)) : nullptr;
    hc = reinterpret_cast<__nv_bfloat16*>(take(2 * Ppad * Dp));
    unit = has_unit ? reinterpret_cast<float*>(take(4 * Ppad * Dp)) : nullptr;
    bytes = at;
  }
};

// ---- before the forward -----------------------------------------------------------------------------
// Blocks 0..row_blocks-1 put the rows whose target counts one behind the other (in their order), as bf16 with zero columns up to Dp.
// The remaining blocks copy the bias with -inf behind V.  Every row block counts the targets before its own itself, from the start of its
// stretch of kPrepStretch rows: up to that many rows a few hundred KB in L2, cheaper than another launch.  More rows have their stretches
// counted by a kernel in front, so that the reading grows with the rows and not with their square (a call with all of its rows ignored:
// 65537 rows 61 us without that kernel and 69 with it, 450563 rows 449 and 295 us, 16 M rows 294 and 10 ms).  A block takes 32 to 512 rows, so that
// two blocks per SM share the copying (4096 rows of 512: 39 us with 512 rows a block).
constexpr int kPrepThreads = 512;
constexpr int64_t kPrepStretch = 65536;  // a multiple of every block's rows

struct PrepParams {
  const void* h;
  int64_t h_row, h_col;  // strides
  int h_fp32, vec;
  const void* targets;
  int64_t t_stride, ignore;
  int t_int32;
  int P, V, D, Dp;
  FsState st;
  float* loss;   // [P] without a reduction, one value with it
  int reduction;
  const void* bias_in;
  int64_t bias_stride;
  int bias_bf16;
  int rows;  // of a block: a multiple of 32
  int row_blocks;
  int64_t* stretches;  // targets of every whole stretch (as fs_target_kind sums them), or null: there is only one
  int gave_up;  // what FS_GAVE_UP starts at
};

__device__ __forceinline__ int64_t fs_target(int64_t i, const PrepParams& p) {
  return p.t_int32 ? int64_t(reinterpret_cast<const int*>(p.targets)[i * p.t_stride]) : reinterpret_cast<const int64_t*>(p.targets)[i * p.t_stride];
}
// 0 ignored, 1 counts, 1 << 32 outside the classes (so that a sum counts both)
__device__ __forceinline__ int64_t fs_target_kind(int64_t t, const PrepParams& p) { return t == p.ignore ? 0 : (t < 0 || t >= p.V ? int64_t(1) << 32 : 1); }

// one block per stretch
__global__ void __launch_bounds__(kPrepThreads) full_softmax_count_kernel(const PrepParams p) {
  __shared__ int64_t sums[kPrepThreads / 32];
  const int64_t begin = int64_t(blockIdx.x) * kPrepStretch, end = min(begin + kPrepStretch, int64_t(p.P));
  int64_t n = 0;
  for (int64_t i = begin + threadIdx.x; i < end; i += kPrepThreads) n += fs_target_kind(fs_target(i, p), p);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) n += sums[w];
    p.stretches[blockIdx.x] = n;
  }
}

__global__ void __launch_bounds__(kPrepThreads) full_softmax_prep_kernel(const PrepParams p) {
  fs_let_next();
  if (int(blockIdx.x) >= p.row_blocks) {
    const int64_t vpad = (int64_t(p.V) + kFsTile - 1) / kFsTile * kFsTile;
    for (int64_t v = int64_t(blockIdx.x - p.row_blocks) * kPrepThreads + threadIdx.x; v < vpad; v += int64_t(gridDim.x - p.row_blocks) * kPrepThreads)
      p.st.bias[v] = v >= p.V        ? -INFINITY
                     : p.bias_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias_in)[v * p.bias_stride])
                                   : reinterpret_cast<const float*>(p.bias_in)[v * p.bias_stride];
    return;
  }
  constexpr int kWarps = kPrepThreads / 32;
  __shared__ int64_t counts[kWarps], befores[kWarps];
  __shared__ int slots[kPrepThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t begin = int64_t(blockIdx.x) * p.rows, row = int(threadIdx.x) < p.rows ? begin + threadIdx.x : p.P;  // P: no row
  int64_t before = 0;
  const int64_t stretch = p.stretches != nullptr ? begin / kPrepStretch : 0;
  for (int64_t i = threadIdx.x; i < stretch; i += kPrepThreads) before += p.stretches[i];
  for (int64_t i = stretch * kPrepStretch + threadIdx.x; i < begin; i += kPrepThreads) before += fs_target_kind(fs_target(i, p), p);
  const int64_t t = row < p.P ? fs_target(row, p) : p.ignore;
  const int64_t kind = fs_target_kind(t, p);
  const uint32_t mine = __ballot_sync(0xffffffffu, kind == 1), bad = __ballot_sync(0xffffffffu, kind > 1);
  const int in_warp = __popc(mine & ((1u << lane) - 1));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) {
    counts[warp] = __popc(mine) + (int64_t(__popc(bad)) << 32);
    befores[warp] = before;
  }
  __syncthreads();
  int64_t first = 0, total = 0, block_total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    total += befores[w];
    block_total += counts[w];
    if (w < warp) first += counts[w];
  }
  const int at = kind == 1 ? int(total & 0x7fffffff) + int(first & 0x7fffffff) + in_warp : -1;
  slots[threadIdx.x] = at;
  if (row < p.P) {
    p.st.slot[row] = at;
    if (at >= 0) {
      p.st.target[at] = int(t);
      p.st.orig[at] = int(row);
    } else if (p.reduction == 0) {
      p.loss[row] = kind > 1 ? __int_as_float(0x7fc00000) : 0.f;
    }
    if (kind > 1) atomicCAS(&g_fs_error, 0, FS_ERR_TARGET);
  }
  if (row < p.P && row % kFsTile == 0) p.st.counters[FS_COUNTERS + row / kFsTile] = 0;
  __syncthreads();
  const bool last = int(blockIdx.x) == p.row_blocks - 1;
  const int n = int((total + block_total) & 0x7fffffff), padded = (n + kFsTile - 1) / kFsTile * kFsTile;
  if (last) {
    if (threadIdx.x == 0) {
      const int n_bad = int((total + block_total) >> 32);
      p.st.counters[FS_N_VALID] = n;
      p.st.counters[FS_N_BAD] = n_bad;
      p.st.counters[FS_JOINED] = 0;
      p.st.counters[FS_FAR] = 0;
      p.st.counters[FS_GAVE_UP] = p.gave_up;
      if (p.reduction != 0 && n == 0) *p.loss = n_bad > 0 ? __int_as_float(0x7fc00000) : 0.f;
    }
    if (n + int(threadIdx.x) < padded) p.st.target[n + threadIdx.x] = -1;
  }
  const int vecs = p.Dp / 8;
  const int rows = int(min(int64_t(p.rows), p.P - begin));
  // eight columns at a time
  for (int i = threadIdx.x; i < rows * vecs; i += kPrepThreads) {
    const int r = i / vecs, c = (i - r * vecs) * 8, to = slots[r];
    if (to < 0) continue;
    uint4 o;
    if (p.vec) {
      o = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.h) + (begin + r) * p.h_row + c);
    } else {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t e = (begin + r) * p.h_row + int64_t(c + k) * p.h_col;
        v[k] = c + k < p.D ? (p.h_fp32 ? reinterpret_cast<const float*>(p.h)[e] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.h)[e])) : 0.f;
      }
      o = make_uint4(fs_pack(v[0], v[1]), fs_pack(v[2], v[3]), fs_pack(v[4], v[5]), fs_pack(v[6], v[7]));
    }
    *reinterpret_cast<uint4*>(p.st.hc + int64_t(to) * p.Dp + c) = o;
  }
  if (last)
    for (int i = threadIdx.x; i < (padded - n) * vecs; i += kPrepThreads) *reinterpret_cast<uint4*>(p.st.hc + int64_t(n) * p.Dp + int64_t(i) * 8) = make_uint4(0, 0, 0, 0);
}

// ---- after the forward: join the splits of every row --------------------------------------------------
// One block per row: the factors of its item's parts (to the highest of their references) go to shared memory, then the threads walk (group of parts, 4 columns).  The
// block that finishes a tile of rows last adds up their losses, and the last of those the tiles', in a fixed order.
constexpr int kJoinThreads = 128;
static_assert(kJoinThreads == kFsTile, "a tile's losses are added up by one block, a row per thread");

struct JoinParams {
  FsState st;
  int V, D, grid, pieces, reduction;
  const float* part_acc;
  const float2* part_m;
  const float* part_l;
  const float* zt;
  float* loss_c;     // [Ppad]
  float* tile_loss;  // [Ppad / 128]
  const __nv_bfloat16* W;
  int64_t ldw;
  float* loss;
};

template <bool ACC>
__global__ void __launch_bounds__(kJoinThreads) full_softmax_join_kernel(const JoinParams p) {
  extern __shared__ __align__(16) float js[];  // [slots of an item] weights, then [threads * 4] partial sums
  fs_after();
  const int n = p.st.counters[FS_N_VALID], n_bad = p.st.counters[FS_N_BAD], row = blockIdx.x;
  const int padded = (n + kFsTile - 1) / kFsTile * kFsTile;
  if (row >= padded) return;
  __shared__ float red[kJoinThreads / 32];
  __shared__ float2 refs[kJoinThreads / 32];
  __shared__ int arrived;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto block_sum = [&](float v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  };
  if (row >= n) {  // a streamed row of zeros: exp(0 - inf) = 0
    if (threadIdx.x == 0) {
      p.st.lse2[row] = INFINITY;
      p.st.lbase[row] = 0.f;
    }
    return;
  }
  const float z = p.zt[row];
  {
    const FsSchedule sc(n, p.V, p.pieces, p.grid);
    const int x = row / kFsTile, r128 = row % kFsTile, whole = sc.whole * p.grid;
    // the slots of an item: count of them from the first
    auto slots = [&](int item, int& first) {
      if (item < whole) {
        first = item;
        return 1;
      }
      const int rel = item - whole, c0 = sc.first_run(rel);
      first = item + c0;
      return sc.last_run(rel) - c0 + 1;
    };
    int first, count = slots(x, first);
    auto load_ref = [&](int64_t at) {
      const float2 v = p.part_m[at];
      FsRef r;
      r.k = v.x;
      r.base = v.y;
      return r;
    };
    FsRef m;
    float l = 0.f;
    for (int s = threadIdx.x; s < 2 * count; s += kJoinThreads) {
      const int64_t at = (int64_t(first) * 2 + s) * kFsTile + r128;
      const FsRef ms = load_ref(at);
      const float ls = p.part_l[at];
      const FsRef mn = fs_higher(m, ms);
      if (mn.k != -INFINITY) l = l * fs_factor(m, mn) + ls * fs_factor(ms, mn);
      else l += ls;
      m = mn;
    }
    const FsRef mine = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      FsRef other;
      other.k = __shfl_xor_sync(0xffffffffu, m.k, o);
      other.base = __shfl_xor_sync(0xffffffffu, m.base, o);
      m = fs_higher(m, other);
    }
    if (lane == 0) refs[warp] = make_float2(m.k, m.base);
    __syncthreads();
    m = FsRef();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) {
      FsRef other;
      other.k = refs[w].x;
      other.base = refs[w].y;
      m = fs_higher(m, other);
    }
    if (m.k == -INFINITY) m.k = 0.f;  // no terms: every factor is 0
    l = block_sum(mine.k == -INFINITY ? l : l * fs_factor(mine, m));
    // others' log sum (base + a2 in base 2) and the target's score z: d = others - z, lse = max + log(1 + e^-|d|)
    const float a2 = m.k + log2f(l), d = fmaf(a2, kLn2, m.base - z), d2 = d * kLog2e;
    const float tail = log1pf(exp2f(-fabsf(d2)));
    const float w = d > 0.f ? 1.f / (1.f + exp2f(-d2)) : exp2f(d2) / (1.f + exp2f(d2));  // 1 - p_t
    if (threadIdx.x == 0) {
      const float loss = p.st.counters[FS_GAVE_UP] != 0 ? __int_as_float(0x7fc00000) : d != d ? d : (d > 0.f ? d : 0.f) + tail;
      const float base = d > 0.f ? m.base : (fabsf(z) < kFar ? 0.f : z);
      p.st.lse2[row] = (d > 0.f ? a2 : (z - base) * kLog2e) + tail * kLog2e;
      p.st.lbase[row] = base;
      if (base != 0.f) p.st.counters[FS_FAR] = 1;  // every writer's value is the same
      p.st.wex[row] = w;
      if (p.reduction == 0) p.loss[p.st.orig[row]] = loss;
      else p.loss_c[row] = loss;
    }
    if constexpr (ACC) {
      float4* buf = reinterpret_cast<float4*>(js + ((p.grid + 7) & ~3));
      const float inv = l > 0.f ? w / l : (l == 0.f ? 0.f : l);
      const int64_t t = p.st.target[row];
      const int acc_width = min(p.D, kFsAcc);
      for (int piece = 0; piece < p.pieces; ++piece) {
        // every piece was cut on its own
        if (piece > 0) count = slots(piece * sc.tx + x, first);
        __syncthreads();
        for (int s = threadIdx.x; s < count; s += kJoinThreads) js[s] = fs_factor(load_ref((int64_t(first) + s) * 2 * kFsTile + r128), m);
        __syncthreads();
        const int vecs = (min(p.D - piece * kFsAcc, kFsAcc)) / 4;  // at most 64
        int lanes = 1;
        while (lanes < vecs) lanes <<= 1;
        const int groups = kJoinThreads / lanes, g = threadIdx.x / lanes, c = threadIdx.x % lanes;
        float4 s4 = f4zero();
        if (c < vecs)
          for (int s = g; s < count; s += groups) {
            const float4 v = *reinterpret_cast<const float4*>(p.part_acc + ((int64_t(first) + s) * kFsTile + r128) * acc_width + c * 4);
            const float f = js[s];
            s4.x += f * v.x;
            s4.y += f * v.y;
            s4.z += f * v.z;
            s4.w += f * v.w;
          }
        buf[threadIdx.x] = s4;
        __syncthreads();
        if (g == 0 && c < vecs) {
          for (int k = 1; k < min(groups, count); ++k) {
            const float4 v = buf[k * lanes + c];
            s4.x += v.x;
            s4.y += v.y;
            s4.z += v.z;
            s4.w += v.w;
          }
          const int col = piece * kFsAcc + c * 4;
          const float4 wt = Vec4<__nv_bfloat16>::load(p.W + t * p.ldw + col);
          *reinterpret_cast<float4*>(p.st.unit + int64_t(row) * p.D + col) =
              make_float4(s4.x * inv - w * wt.x, s4.y * inv - w * wt.y, s4.z * inv - w * wt.z, s4.w * inv - w * wt.w);
        }
      }
    }
  }
  if (p.reduction == 0) return;
  auto last_of = [&](int* counter, int count) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      arrived = atomicAdd(counter, 1);
    }
    __syncthreads();
    if (arrived != count - 1) return false;
    __threadfence();
    return true;
  };
  const int tile = row / kFsTile;
  const int in_tile = min(kFsTile, n - tile * kFsTile), tiles = padded / kFsTile;
  if (in_tile > 1 && !last_of(p.st.counters + FS_COUNTERS + tile, in_tile)) return;
  float s = block_sum(int(threadIdx.x) < in_tile ? __ldcg(p.loss_c + tile * kFsTile + threadIdx.x) : 0.f);
  if (tiles > 1) {
    if (threadIdx.x == 0) p.tile_loss[tile] = s;
    if (!last_of(p.st.counters + FS_JOINED, tiles)) return;
    s = 0.f;
    for (int k = threadIdx.x; k < tiles; k += kJoinThreads) s += __ldcg(p.tile_loss + k);
    s = block_sum(s);
  }
  if (threadIdx.x == 0) *p.loss = n_bad > 0 ? __int_as_float(0x7fc00000) : (p.reduction == 1 ? s / float(n) : s);
}

// ---- backward ---------------------------------------------------------------------------------------------
// upstream gradients of the compacted rows (no reduction), zero behind the last
__global__ void full_softmax_gcol_kernel(FsState st, const float* __restrict__ dloss, int64_t stride, float* __restrict__ gcol) {
  const int n = st.counters[FS_N_VALID], i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < (n + kFsTile - 1) / kFsTile * kFsTile) gcol[i] = i < n ? dloss[st.orig[i] * stride] : 0.f;
}

struct FinishParams {
  FsState st;
  int P, V, D, Dp, grid, pieces, per_row, mean;
  const float* dloss;
  int64_t dl_stride;
  const float* part_acc;  // or null: dW was written by the main kernel
  const float* part_l;
  void* dh;               // [P, D] or null
  void* dw;               // [dw_rows, Dp]
  int64_t dw_rows;        // V, or 0
  void* db;               // [V] or null
  int db_bf16;
};

template <typename T>
__device__ __forceinline__ void fs_store8(T* o, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(o) = make_uint4(fs_pack(v[0], v[1]), fs_pack(v[2], v[3]), fs_pack(v[4], v[5]), fs_pack(v[6], v[7]));
  } else {
    reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// dh = g * unit at the rows' own places; the splits of dW and db joined in their order
template <typename TH, typename TW>
__global__ void __launch_bounds__(256) full_softmax_finish_kernel(const FinishParams p) {
  fs_after();
  const int n = p.st.counters[FS_N_VALID], vecs = p.Dp / 8;
  const bool gave_up = p.st.counters[FS_GAVE_UP] != 0;  // in this pass or in the forward: what the blocks left is not to be used
  const int64_t step = int64_t(gridDim.x) * blockDim.x, me = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const float g_all = p.per_row ? 1.f : *p.dloss / (p.mean ? float(max(n, 1)) : 1.f);
  if (p.dh != nullptr) {
    for (int64_t i = me; i < int64_t(p.P) * vecs; i += step) {
      const int64_t row = i / vecs;
      const int c = int(i - row * vecs) * 8, at = p.st.slot[row];
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
      if (at >= 0) {
        const float g = p.per_row ? p.dloss[row * p.dl_stride] : g_all;
        const float4* u = reinterpret_cast<const float4*>(p.st.unit + int64_t(at) * p.Dp + c);
        const float4 a = u[0], b = u[1];
        v[0] = a.x * g; v[1] = a.y * g; v[2] = a.z * g; v[3] = a.w * g;
        v[4] = b.x * g; v[5] = b.y * g; v[6] = b.z * g; v[7] = b.w * g;
        if (gave_up) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = __int_as_float(0x7fc00000);
        }
      }
      TH* o = reinterpret_cast<TH*>(p.dh) + row * p.D + c;
      if (p.D == p.Dp) {
        fs_store8(o, v);
      } else {
        for (int k = 0; k < 8 && c + k < p.D; ++k) o[k] = TH(v[k]);
      }
    }
  }
  if (gave_up) {
    const float nan = __int_as_float(0x7fc00000);
    const float v[8] = {nan, nan, nan, nan, nan, nan, nan, nan};
    for (int64_t i = me; i < p.dw_rows * vecs; i += step) fs_store8(reinterpret_cast<TW*>(p.dw) + i * 8, v);
    if (p.db != nullptr)
      for (int64_t i = me; i < p.V; i += step) {
        if (p.db_bf16) reinterpret_cast<__nv_bfloat16*>(p.db)[i] = __float2bfloat16(nan);
        else reinterpret_cast<float*>(p.db)[i] = nan;
      }
    return;
  }
  if (p.part_acc == nullptr && p.db == nullptr) return;
  const FsSchedule sc(p.V, n, p.pieces, p.grid);
  const int whole = sc.whole * p.grid;
  if (p.part_acc != nullptr) {
    // items left over that were cut (the others were written by the main kernel)
    const int acc_width = min(p.Dp, kFsAcc), wv = acc_width / 8;
    for (int64_t i = me; i < int64_t(sc.rest) * kFsTile * wv; i += step) {
      const int c = int(i % wv) * 8, r128 = int(i / wv % kFsTile), rel = int(i / wv / kFsTile);
      const int c0 = sc.first_run(rel), c1 = sc.last_run(rel), item = whole + rel, x = item % sc.tx, piece = item / sc.tx;
      const int64_t row = int64_t(x) * kFsTile + r128;
      if (c0 == c1 || row >= p.V || piece * kFsAcc + c >= p.Dp) continue;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
      for (int s = c0; s <= c1; ++s) {
        const float4* x4 = reinterpret_cast<const float4*>(p.part_acc + (int64_t(rel + s) * kFsTile + r128) * acc_width + c);
        const float4 a = x4[0], b = x4[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= g_all;
      fs_store8(reinterpret_cast<TW*>(p.dw) + row * p.Dp + piece * kFsAcc + c, v);
    }
  }
  if (p.db != nullptr)
    for (int64_t v = me; v < p.V; v += step) {
      const int item = int(v / kFsTile), r128 = int(v % kFsTile);
      int first = item, count = 1;
      if (item >= whole) {
        const int c0 = sc.first_run(item - whole);
        first = item + c0;
        count = sc.last_run(item - whole) - c0 + 1;
      }
      float s = 0.f;
      for (int k = 0; k < 2 * count; ++k) s += p.part_l[(int64_t(first) * 2 + k) * kFsTile + r128];
      s *= g_all;
      if (p.db_bf16) reinterpret_cast<__nv_bfloat16*>(p.db)[v] = __float2bfloat16(s);
      else reinterpret_cast<float*>(p.db)[v] = s;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------
static int fs_grid(const at::Device& dev) { return at::cuda::getDeviceProperties(dev.index())->multiProcessorCount; }

template <int MODE, bool BIAS, bool ROWG>
static void fs_launch(const CUtensorMap& tx, const CUtensorMap& ty, const FsParams& p, int device) {
  auto kernel = full_softmax_kernel<MODE, BIAS, ROWG>;
  static bool set[64] = {};  // the attribute is per kernel and device; setting it twice is harmless
  if (device >= 64 || !set[device]) {
    TRB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFsSmem));
    if (device < 64) set[device] = true;
  }
  fs_launch_next(kernel, p.grid, kFsThreads, kFsSmem, at::cuda::getCurrentCUDAStream(), tx, ty, p);
}

static void fs_shape(FsParams& p, int64_t V, int64_t D, bool acc) {
  p.V = int(V);
  p.D = int(D);
  p.kb = int((D + 63) / 64);
  p.x_resident = p.kb <= 8;       // with up to 8 of 14 slots for X the ring keeps three units of two blocks
  p.hold = acc && p.kb <= 4;      // two tiles of four blocks, X and one more unit fit
}

constexpr int64_t kFsMaxRows = (int64_t(1) << 31) - 2 * kFsTile;

static void fs_check_weight(const at::Tensor& w) {
  TORCH_CHECK_VALUE(w.is_cuda() && w.scalar_type() == at::kBFloat16 && w.dim() == 2 && w.stride(1) == 1 && w.size(0) >= 1 && w.size(0) < kFsMaxRows,
                    "full_softmax: the weight is a bf16 [V, D] matrix with contiguous rows");
  TORCH_CHECK_VALUE(w.size(1) >= 8 && w.size(1) % 8 == 0 && w.size(1) <= kFsMaxD && w.stride(0) % 8 == 0 && w.stride(0) >= w.size(1) &&
                        reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
                    "full_softmax: D and the row pitch of the weight are multiples of 8 (D at most ", kFsMaxD, "), its rows start on 16 bytes");
}

// h [P, D] bf16 or fp32 (any strides), weight [V, Dp] bf16 with Dp = D rounded up to 8 (zero columns behind D), targets [P] int64 or
// int32, bias [V] fp32 or bf16 or none.  reduction: 0 none, 1 mean, 2 sum.  grad: 0 loss only, 1 prepare the backward of W and b, 2 of h
// too.  Returns the loss and the state for the backward.  gave_up: not 0 gives what a call gives in which a block gave up its wait.
std::tuple<at::Tensor, at::Tensor> full_softmax_fwd(const at::Tensor& h, const at::Tensor& weight, const at::Tensor& targets, const c10::optional<at::Tensor>& bias,
                                                    int64_t ignore_index, int64_t reduction, int64_t grad, int64_t gave_up) {
  fs_check_weight(weight);
  TORCH_CHECK_VALUE(h.is_cuda() && h.dim() == 2 && (h.scalar_type() == at::kBFloat16 || h.scalar_type() == at::kFloat), "full_softmax: h is a bf16 or fp32 CUDA tensor [P, D]");
  TORCH_CHECK_VALUE(targets.is_cuda() && targets.dim() == 1 && (targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt) && targets.size(0) == h.size(0),
                    "full_softmax: targets is an int32 or int64 [P]");
  TORCH_CHECK_VALUE(h.device() == weight.device() && h.device() == targets.device(), "full_softmax: operands on different devices");
  TORCH_CHECK_VALUE(reduction >= 0 && reduction <= 2 && grad >= 0 && grad <= 2, "full_softmax: unknown reduction or gradient level");
  const int64_t P = h.size(0), D = h.size(1), V = weight.size(0), Dp = weight.size(1);
  TORCH_CHECK_VALUE(P < kFsMaxRows && D >= 1 && D <= Dp && Dp - D < 8, "full_softmax: h and weight differ in width");
  const bool has_bias = bias.has_value() && bias->defined();
  if (has_bias)
    TORCH_CHECK_VALUE(bias->is_cuda() && bias->device() == h.device() && (bias->scalar_type() == at::kFloat || bias->scalar_type() == at::kBFloat16) && bias->dim() == 1 &&
                          bias->size(0) == V,
                      "full_softmax: bias is an fp32 or bf16 [V]");
  c10::cuda::CUDAGuard guard(h.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t Ppad = (P + kFsTile - 1) / kFsTile * kFsTile, Vpad = (V + kFsTile - 1) / kFsTile * kFsTile;
  const auto f32 = h.options().dtype(at::kFloat);
  const bool acc = grad == 2;
  at::Tensor state = at::empty({FsState(nullptr, P, V, Dp, has_bias, acc).bytes}, h.options().dtype(at::kByte));
  const FsState st(state.data_ptr(), P, V, Dp, has_bias, acc);
  at::Tensor loss = reduction == 0 ? at::empty({P}, f32) : at::empty({}, f32);
  if (P == 0) {
    state.zero_();
    if (reduction != 0) loss.zero_();
    return {loss, state};
  }
  const int grid = fs_grid(h.device());
  const int pieces = acc ? int((Dp + kFsAcc - 1) / kFsAcc) : 1;
  const int64_t prows = (Ppad / kFsTile * pieces + grid) * kFsTile, n_acc = acc ? prows * std::min<int64_t>(Dp, kFsAcc) : 0;  // rows of all slots
  const int64_t n_stretch = P > kPrepStretch ? (P + kPrepStretch - 1) / kPrepStretch : 0;
  // accumulators, references, sums, targets' scores, losses, counts of the stretches (on 8 bytes), losses of the tiles
  at::Tensor part = at::empty({n_acc + 6 * prows + 2 * Ppad + 2 * n_stretch + Ppad / kFsTile}, f32);
  float* part_acc = part.data_ptr<float>();
  float2* part_m = reinterpret_cast<float2*>(part_acc + n_acc);
  float* part_l = part_acc + n_acc + 4 * prows;
  float* zt = part_l + 2 * prows;
  float* loss_c = zt + Ppad;
  int64_t* stretches = n_stretch > 0 ? reinterpret_cast<int64_t*>(loss_c + Ppad) : nullptr;
  float* tile_loss = loss_c + Ppad + 2 * n_stretch;
  {
    int rows = 32;
    while (rows < kPrepThreads && int64_t(rows) * 2 * grid < P) rows *= 2;
    const int row_blocks = int((P + rows - 1) / rows);
    const int bias_blocks = has_bias ? int(std::min<int64_t>((Vpad + kPrepThreads - 1) / kPrepThreads, 2 * grid)) : 0;
    const bool fp32 = h.scalar_type() == at::kFloat;
    const bool vec = !fp32 && D == Dp && h.stride(1) == 1 && h.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(h.data_ptr()) % 16 == 0;
    const PrepParams q{h.data_ptr(), h.stride(0), h.stride(1), fp32, vec, targets.data_ptr(), targets.stride(0), ignore_index, targets.scalar_type() == at::kInt,
                       int(P), int(V), int(D), int(Dp), st, loss.data_ptr<float>(), int(reduction), has_bias ? bias->data_ptr() : nullptr, has_bias ? bias->stride(0) : 0,
                       has_bias && bias->scalar_type() == at::kBFloat16, rows, row_blocks, stretches, gave_up != 0};
    if (n_stretch > 0) {
      full_softmax_count_kernel<<<unsigned(n_stretch), kPrepThreads, 0, stream>>>(q);
      TRB_CUDA_CHECK(cudaGetLastError());
    }
    full_softmax_prep_kernel<<<row_blocks + bias_blocks, kPrepThreads, 0, stream>>>(q);
    TRB_CUDA_CHECK(cudaGetLastError());
  }
  FsParams p{};
  fs_shape(p, V, Dp, acc);
  p.n_valid = st.counters + FS_N_VALID;
  p.gave_up = st.counters + FS_GAVE_UP;
  p.grid = grid;
  p.target = st.target;
  p.bias = st.bias;
  p.part_acc = part_acc;
  p.part_m = part_m;
  p.part_l = part_l;
  p.zt = zt;
  const CUtensorMap tx = make_tmap(st.hc, Ppad, Dp, Dp, 64, kFsTile);
  const CUtensorMap ty = make_tmap(weight.data_ptr(), V, Dp, weight.stride(0), 64, kFsTile);
  const int dev = h.device().index();
  if (acc) has_bias ? fs_launch<FS_FWD, true, false>(tx, ty, p, dev) : fs_launch<FS_FWD, false, false>(tx, ty, p, dev);
  else has_bias ? fs_launch<FS_LSE, true, false>(tx, ty, p, dev) : fs_launch<FS_LSE, false, false>(tx, ty, p, dev);
  const JoinParams j{st, int(V), int(Dp), grid, pieces, int(reduction), part_acc, part_m, part_l, zt, loss_c, tile_loss, reinterpret_cast<const __nv_bfloat16*>(weight.data_ptr()),
                     weight.stride(0), loss.data_ptr<float>()};
  const int smem = (grid + 8) * 4 + kJoinThreads * 16;
  if (acc) fs_launch_next(full_softmax_join_kernel<true>, unsigned(Ppad), kJoinThreads, smem, stream, j);
  else fs_launch_next(full_softmax_join_kernel<false>, unsigned(Ppad), kJoinThreads, 0, stream, j);
  return {loss, state};
}

// dloss: fp32, [P] for reduction 0, a scalar otherwise.  Outputs that are not wanted come back empty.  dh [P, D] in bf16 or fp32,
// dW [V, Dp] in bf16 or fp32, db [V] in fp32 or bf16.
std::tuple<at::Tensor, at::Tensor, at::Tensor> full_softmax_bwd(const at::Tensor& dloss, const at::Tensor& weight, const at::Tensor& state, int64_t P, int64_t D, bool has_bias,
                                                                int64_t reduction, bool has_unit, bool want_h, bool want_w, bool want_b, bool dh_fp32, bool dw_fp32, bool db_fp32) {
  fs_check_weight(weight);
  const int64_t V = weight.size(0), Dp = weight.size(1);
  const at::Device device = weight.device();
  TORCH_CHECK(P >= 0 && P < kFsMaxRows && D >= 1 && D <= Dp && Dp - D < 8 && reduction >= 0 && reduction <= 2);
  TORCH_CHECK(dloss.device() == device && dloss.scalar_type() == at::kFloat && (reduction == 0 ? dloss.dim() == 1 && dloss.size(0) == P : dloss.numel() == 1),
              "full_softmax_bwd: the upstream gradient is fp32, [P] without a reduction and one value with it");
  TORCH_CHECK((!want_b || has_bias) && (!want_h || has_unit));
  TORCH_CHECK(state.device() == device && state.scalar_type() == at::kByte && state.is_contiguous() && state.numel() == FsState(nullptr, P, V, Dp, has_bias, has_unit).bytes,
              "full_softmax_bwd: not the state of this forward");
  const FsState st(state.data_ptr(), P, V, Dp, has_bias, has_unit);
  c10::cuda::CUDAGuard guard(device);
  auto stream = at::cuda::getCurrentCUDAStream();
  const auto f32 = weight.options().dtype(at::kFloat);
  const bool main = want_w || want_b;
  at::Tensor dh = at::empty({want_h ? P : 0, D}, dh_fp32 ? f32 : weight.options());
  at::Tensor dw = at::empty({main ? V : 0, Dp}, dw_fp32 ? f32 : weight.options());  // the kernel that sums db computes dW on the way
  at::Tensor db = at::empty({want_b ? V : 0}, db_fp32 ? f32 : weight.options());
  if (P == 0) {
    dw.zero_();
    db.zero_();
    return {dh, dw, db};
  }
  const int64_t Ppad = (P + kFsTile - 1) / kFsTile * kFsTile, Vpad = (V + kFsTile - 1) / kFsTile * kFsTile;
  const int grid = fs_grid(device), dev = device.index();
  const bool per_row = reduction == 0, mean = reduction == 1;
  const int pieces = int((Dp + kFsAcc - 1) / kFsAcc);
  const int64_t items = Vpad / kFsTile * pieces, rest = items % grid;
  const bool may_split = main && rest > 0 && Ppad > kFsTile;  // items left over, of more than one tile
  const int64_t n_acc = may_split ? (rest + grid) * kFsTile * std::min<int64_t>(Dp, kFsAcc) : 0, n_l = main && has_bias ? 2 * (items + grid) * kFsTile : 0,
                n_g = main && per_row ? Ppad : 0;
  at::Tensor part = n_acc + n_l + n_g > 0 ? at::empty({n_acc + n_l + n_g}, f32) : at::Tensor();
  float* part_acc = n_acc ? part.data_ptr<float>() : nullptr;
  float* part_l = n_l ? part.data_ptr<float>() + n_acc : nullptr;
  float* gcol = n_g ? part.data_ptr<float>() + n_acc + n_l : nullptr;
  if (main) {
    if (gcol != nullptr) {
      full_softmax_gcol_kernel<<<unsigned((Ppad + 255) / 256), 256, 0, stream>>>(st, dloss.data_ptr<float>(), dloss.stride(0), gcol);
      TRB_CUDA_CHECK(cudaGetLastError());
    }
    FsParams p{};
    fs_shape(p, V, Dp, true);
    p.n_valid = st.counters + FS_N_VALID;
    p.gave_up = st.counters + FS_GAVE_UP;
    p.grid = grid;
    p.target = st.target;
    p.bias = st.bias;
    p.part_acc = part_acc;
    p.part_l = part_l;
    p.lse2 = st.lse2;
    p.lbase = st.lbase;
    p.far = st.counters + FS_FAR;
    p.wex = st.wex;
    p.gcol = gcol;
    p.dloss = dloss.data_ptr<float>();
    p.mean = mean;
    p.dw = dw.data_ptr();
    p.dw_fp32 = dw_fp32;
    const CUtensorMap tx = make_tmap(weight.data_ptr(), V, Dp, weight.stride(0), 64, kFsTile);
    const CUtensorMap ty = make_tmap(st.hc, Ppad, Dp, Dp, 64, kFsTile);
    if (has_bias) per_row ? fs_launch<FS_BWD, true, true>(tx, ty, p, dev) : fs_launch<FS_BWD, true, false>(tx, ty, p, dev);
    else per_row ? fs_launch<FS_BWD, false, true>(tx, ty, p, dev) : fs_launch<FS_BWD, false, false>(tx, ty, p, dev);
  }
  if (want_h || main) {  // (behind every main kernel: it looks whether a block gave up)
    const FinishParams f{st, int(P), int(V), int(D), int(Dp), grid, pieces, per_row, mean, dloss.data_ptr<float>(), per_row ? dloss.stride(0) : 0, part_acc, part_l,
                         want_h ? dh.data_ptr() : nullptr, dw.data_ptr(), main ? V : 0, want_b ? db.data_ptr() : nullptr, !db_fp32};
    const int64_t most = std::max<int64_t>({want_h ? P * (Dp / 8) : 0, n_acc / 8, want_b ? V : 0, 1});
    const unsigned blocks = unsigned(std::min<int64_t>((most + 255) / 256, 16 * grid));
    auto finish = dh_fp32 ? (dw_fp32 ? full_softmax_finish_kernel<float, float> : full_softmax_finish_kernel<float, __nv_bfloat16>)
                          : (dw_fp32 ? full_softmax_finish_kernel<__nv_bfloat16, float> : full_softmax_finish_kernel<__nv_bfloat16, __nv_bfloat16>);
    if (main) {
      fs_launch_next(finish, blocks, 256, 0, stream, f);
    } else {
      finish<<<blocks, 256, 0, stream>>>(f);
      TRB_CUDA_CHECK(cudaGetLastError());
    }
  }
  return {dh, dw, db};
}

// Raises the error word for targets outside [0, classes): calls that no kernel takes report them as the others do, without a look from the host.
__global__ void full_softmax_targets_kernel(const int64_t* __restrict__ targets, int64_t n, int64_t stride, int64_t classes, int64_t ignore) {
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t t = targets[i * stride];
    if (t != ignore && (t < 0 || t >= classes)) atomicCAS(&g_fs_error, 0, FS_ERR_TARGET);
  }
}

void full_softmax_check_targets(const at::Tensor& targets, int64_t classes, int64_t ignore_index) {
  TORCH_CHECK_VALUE(targets.is_cuda() && targets.dim() == 1 && targets.scalar_type() == at::kLong, "full_softmax_check_targets: targets is an int64 [P]");
  if (targets.numel() == 0) return;
  c10::cuda::CUDAGuard guard(targets.device());
  const unsigned blocks = unsigned(std::min<int64_t>((targets.numel() + 255) / 256, 4 * fs_grid(targets.device())));
  full_softmax_targets_kernel<<<blocks, 256, 0, at::cuda::getCurrentCUDAStream()>>>(targets.data_ptr<int64_t>(), targets.numel(), targets.stride(0), classes, ignore_index);
  TRB_CUDA_CHECK(cudaGetLastError());
}

// non-zero after a launch gave up waiting (1..9) or met a target outside [0, V) (16); reading it synchronises and resets it
int64_t full_softmax_status() {
  int v = 0;
  const int zero = 0;
  TRB_CUDA_CHECK(cudaDeviceSynchronize());
  TRB_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_fs_error, sizeof(int)));
  if (v != 0) TRB_CUDA_CHECK(cudaMemcpyToSymbol(g_fs_error, &zero, sizeof(int)));
  return v;
}

}  // namespace trb

TORCH_LIBRARY_FRAGMENT(trb200, m) {
  m.def("full_softmax_fwd(Tensor h, Tensor weight, Tensor targets, Tensor? bias, int ignore_index, int reduction, int grad, int gave_up=0) -> (Tensor, Tensor)");
  m.def("full_softmax_bwd(Tensor dloss, Tensor weight, Tensor state, int P, int D, bool has_bias, int reduction, bool has_unit, bool want_h, bool want_w, bool want_b, "
        "bool dh_fp32, bool dw_fp32, bool db_fp32) -> (Tensor, Tensor, Tensor)");
  m.def("full_softmax_check_targets(Tensor targets, int classes, int ignore_index) -> ()");
  m.def("full_softmax_status() -> int");
}

TORCH_LIBRARY_IMPL(trb200, CUDA, m) {
  m.impl("full_softmax_fwd", &trb::full_softmax_fwd);
  m.impl("full_softmax_bwd", &trb::full_softmax_bwd);
  m.impl("full_softmax_check_targets", &trb::full_softmax_check_targets);
}

TORCH_LIBRARY_IMPL(trb200, CompositeExplicitAutograd, m) { m.impl("full_softmax_status", &trb::full_softmax_status); }
