// feed_forward_tensor.cu -- the feed-forward block's products of 16-bit types on
// the tensor cores (geo/geo_b200.h section 5).
//
// All products are C = A B in steps of 64 of K. Large ones (PAIR) go over tiles of 256
// rows by 256 columns, on which two blocks on neighbouring multiprocessors work
// (tcgen05 cta_group::2): each copies its own 128 rows of A and half of the columns of
// B, and the first block's instructions multiply for both, 256 x 256 x 16 at a time. 32
// KB copied a block of K, where single blocks copy 48: their way from L2 into shared
// memory is what bounds those (the instructions of the VJP's products waited 28 to 59%
// of their time for data). Up to 128 rows, and where pairs would leave multiprocessors
// idle, single blocks take tiles of 128 rows by BN = 64, 128 or 256 columns.
// One block a multiprocessor, persistent over its tiles, six warps or ten:
//   warp 0   one thread copies tiles of A and B into a ring of stages (TMA,
//            128-byte swizzle, completion on the stage's `full` mbarrier; a pair's on
//            the first block's);
//   warp 1   one thread (a pair's first block's) issues the matrix instructions of a
//            stage (tcgen05.mma) and commits them to the stage's `empty` mbarrier, a
//            tile's last to `ready`; the float32 sums stand in tensor memory, two
//            tiles of BN columns in turn;
//   warps 2-5 (2-9 where there is more to do) take a finished tile out of tensor
//            memory (32 rows a warp), do what belongs to the product (activation, its
//            derivative), round once and write it through shared memory in whole
//            64-byte pieces, while the next tile is multiplied.
// Operands whose sum index is not the adjacent one (weights in the VJP, both sides
// of the weights' cotangents) are copied as they lie, [64 of K][64 values] boxes,
// and read by the matrix instruction as "MN-major": nothing is transposed.
// kGated puts BN / 2 rows of each weight side by side in one B tile, so that gate and
// up of the same hidden values are in one tile of sums; kInput adds both its products
// into one tile, K running through the first pair of operands, then the second.
// Measured: 8192 x 4096 x 12288 bfloat16, gate and up 1.17 ms (1.41 PFLOP/s), down 0.59,
// the VJP to float32 cotangents 5.75 to 6.6 ms with 7.4 TFLOP, its last product with 96% of
// the tensor cycles: the board's power bounds them (1.3 GHz). The VJP's first product
// reads two arrays more and writes six: 1.1 ms where its multiplications take 0.6.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

constexpr int kBM = 128, kBK = 64;
// Warps that take the sums out. The VJP's first product reads two more arrays and
// writes up to six; float32 results of two-term operands are summed up in registers.
constexpr int epilogue_warps(int kind, bool twice) { return kind == kHidden || twice ? 8 : 4; }
// Blocks of K that are summed in tensor memory in one go, where the results are float32
// or two-term: the tensor cores cut where float32 arithmetic rounds, which takes 2e-8 of
// the size off with each 16 of K (1.8e-5 over 8192 rows; five times that where all
// products have one sign; float16 values below 2^-14 count as such of 2^-14 there, so that
// sums of those alone are cut at 2^-39 of the other operand's size). The parts are added up in
// registers, rounded to nearest. VJP of 8192 x 4096 x 12288 to float32 cotangents, this
// many blocks, a weight's cotangent's error and the time in calls one after another:
//   bfloat16  16 blocks 4.1e-6, 6.08 ms; 8 blocks 3.0e-6, 6.1 to 6.3; 4 blocks 2.6e-6, 6.5
//   float16   16 blocks 3.5e-6, 7.0 ms;  8 blocks 1.8e-6, 7.1;        4 blocks 1.0e-6, 7.1
// What two terms of bfloat16 lose is 2.2e-6 of it, of float16 nothing: it takes shorter parts.
template <typename T>
constexpr int kChunk = std::is_same_v<T, __half> ? 4 : 8;
// Blocks of K that are summed up in tensor memory in one go at most, by more parts of K
// where there are more: sums of like signs lose 1.0e-7 with each 16 of K (of random signs
// less), so that these leave 1.0e-4 (float16) and 2.1e-4, a fifth and a nineteenth of the
// result's own rounding. 65536 of K in one go left 4.2e-4.
constexpr int longest(uint32_t type) { return type == GEO_B200_F16 ? 256 : 512; }
constexpr uint32_t bytes_a(bool twice) { return (twice ? 2 : 1) * kBM * kBK * 2; }
constexpr uint32_t bytes_b(int bn) { return (uint32_t)bn * kBK * 2; }
// A warp's shared memory: 32 rows of 64 bytes, 16 more bytes a row to keep banks apart.
// kHidden: two of those for what it reads, and two of 32 x 64 bytes (swizzled, so that a
// copy of the whole can take them out) for what it writes.
constexpr uint32_t kRows = 32 * 80, kBox = 32 * 64;
constexpr uint32_t staging_of(int kind) { return kind == kHidden ? 2 * kBox + 2 * kRows : kRows; }
constexpr uint32_t kSharedMost = 227 * 1024;
// A block's part of a stage.
constexpr uint32_t stage_bytes(int bn, bool twice, bool pair) { return bytes_a(twice) + bytes_b(bn) / (pair ? 2 : 1); }
constexpr int stages_of(int kind, int bn, bool twice, bool pair) {
    const int n = (int)((kSharedMost - 1024 - epilogue_warps(kind, twice) * staging_of(kind) - 512) /
                        stage_bytes(bn, twice, pair));
    return n > 8 ? 8 : n;
}
constexpr uint32_t shared_bytes(int kind, int bn, bool twice, bool pair) {
    return 1024 + stages_of(kind, bn, twice, pair) * stage_bytes(bn, twice, pair) +
           epilogue_warps(kind, twice) * staging_of(kind);
}

// Rows of a box of A [M][K].
__host__ __device__ constexpr int box_rows(int m) { return m < kBM ? (m + 7) / 8 * 8 : kBM; }

struct Maps {
    CUtensorMap a[3], b[3], low[3];
    CUtensorMap out[6];  // kHidden: out[0], out_low[0], out[1], ...
};

__device__ __forceinline__ void barrier_init(uint32_t barrier, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
// Takes bytes that will not come off what the phase expects.
__device__ __forceinline__ void barrier_excuse(uint32_t barrier, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t barrier) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
}
// The same place of the shared memory of the pair's block `rank`.
__device__ __forceinline__ uint32_t place_of(uint32_t here, uint32_t rank) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
    return there;
}
__device__ __forceinline__ void store_cluster(uint32_t there, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}
__device__ __forceinline__ void barrier_arrive_cluster(uint32_t there) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t barrier, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(barrier), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for the phase, at most `polls` looks; false when it gave up or another warp did.
__device__ __forceinline__ bool barrier_wait(uint32_t barrier, uint32_t parity, uint32_t polls, volatile int *gave_up) {
    for (uint32_t i = 0; i < polls; ++i) {
        if (barrier_try(barrier, parity)) return true;
        if (gave_up != nullptr && *gave_up) return false;
    }
    if (gave_up != nullptr) *gave_up = 1;
    return false;
}

// A box of the tensor to this block's shared memory; `barrier` may be of the pair's first block.
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t barrier) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
            "[%0], [%1, {%2, %3}], [%4];" ::"r"(to),
            "l"(map), "r"(x), "r"(y), "r"(barrier)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                to),
            "l"(map), "r"(x), "r"(y), "r"(barrier)
            : "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled operand. Its eight-row groups are
// 1024 bytes apart; `leading`: bytes between blocks of 64 values (MN-major only).
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t leading) {
    return (uint64_t)((address & 0x3FFFF) >> 4) | (uint64_t)((leading >> 4) & 0x3FFF) << 16 |
           (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 16-bit operands, float32 sums, m x n.
template <typename T>
__device__ __forceinline__ constexpr uint32_t instruction(bool a_mn, bool b_mn, int m, int n) {
    const uint32_t format = std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
    return 1u << 4 | format << 7 | format << 10 | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 |
           (uint32_t)(n / 8) << 17 | (uint32_t)(m / 16) << 24;
}
template <bool PAIR>
__device__ __forceinline__ void multiply(uint32_t sums, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
    if constexpr (PAIR)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(sums),
            "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(sums),
            "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
            : "memory");
}
// Arrives at the barrier (PAIR: of both blocks) once the matrix instructions so far have ended.
template <bool PAIR>
__device__ __forceinline__ void commit_to(uint32_t barrier) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                barrier),
            "h"((unsigned short)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier)
                     : "memory");
}

// 32 columns of this thread's row of the warp's 32 rows of tensor memory.
__device__ __forceinline__ void take_columns(uint32_t address, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// And back: 32 columns of this thread's row.
__device__ __forceinline__ void leave_columns(uint32_t address, const float *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(address),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
        "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
        "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
        : "memory");
}

// Whether rows of this array can be read and written by 16 bytes.
template <typename T>
__device__ __forceinline__ bool by_16(const void *p, size_t stride) {
    return ((uintptr_t)p % 16 | stride * sizeof(T) % 16) == 0;
}

// Writes 64 bytes of this thread's row (rows row0 + lane, columns col0 ...) of an m x n
// array, through the warp's staging.
template <typename O>
__device__ __forceinline__ void put_words(unsigned char *staging, const uint32_t (&words)[16], const OutMatrix &out,
                                          int row0, int col0, int m, int n) {
    constexpr int kVector = 16 / (int)sizeof(O), kWidth = 64 / (int)sizeof(O), kPitch = 80;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *(uint4 *)(staging + lane * kPitch + 16 * j) =
            make_uint4(words[4 * j], words[4 * j + 1], words[4 * j + 2], words[4 * j + 3]);
    __syncwarp();
    if (by_16<O>(out.p, out.stride)) {
        const int c = col0 + lane % 4 * kVector;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 8) {
            const int r = r0 + lane / 4;
            if (row0 + r >= m || c >= n) continue;
            const O *piece = (const O *)(staging + r * kPitch) + lane % 4 * kVector;
            O *to = (O *)out.p + (size_t)(row0 + r) * out.stride + c;
            if (c + kVector <= n) {
                store<O, kVector>(to, load<O, kVector>(piece));
            } else {
                for (int j = 0; c + j < n; ++j) to[j] = piece[j];
            }
        }
    } else {
        for (int r = lane / kWidth; r < 32 && row0 + r < m; r += 32 / kWidth)
            if (col0 + lane % kWidth < n)
                ((O *)out.p)[(size_t)(row0 + r) * out.stride + col0 + lane % kWidth] =
                    ((const O *)(staging + r * kPitch))[lane % kWidth];
    }
    __syncwarp();
}
// Writes 32 columns of 16-bit values of this thread's row as a box of the array that
// `map` describes (columns and rows from col0 and row0), which its ends clip: one copy
// for the warp instead of the loads and stores of put_words. `box`: the next of the
// warp's two boxes, which the copy before the last one has read.
__device__ __forceinline__ void put_box(unsigned char *box, const uint32_t (&words)[16], const CUtensorMap *map, int row0,
                                        int col0) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)  // 64-byte swizzle
        *(uint4 *)(box + lane * 64 + (j ^ (lane >> 1 & 3)) * 16) =
            make_uint4(words[4 * j], words[4 * j + 1], words[4 * j + 2], words[4 * j + 3]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(col0),
                     "r"(row0), "r"(shared_address(box))
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
// Two neighbours as a word of 16-bit values.
template <typename T>
__device__ __forceinline__ uint32_t word_of(float x, float y) {
    Vec<T, 2> v;
    v.set(0, {x, y});
    return v.w[0];
}
// 32 columns, v[from ...].
template <typename O, int COUNT>
__device__ __forceinline__ void put_columns(unsigned char *staging, const float (&v)[COUNT], int from,
                                            const OutMatrix &out, int row0, int col0, int m, int n) {
#pragma unroll
    for (int part = 0; part < (int)sizeof(O) / 2; ++part) {
        if (part > 0 && col0 + 16 >= n) break;
        uint32_t words[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (sizeof(O) == 4)
                words[i] = __float_as_uint(v[from + part * 16 + i]);
            else
                words[i] = word_of<O>(v[from + 2 * i], v[from + 2 * i + 1]);
        }
        put_words<O>(staging, words, out, row0, col0 + part * 16, m, n);
    }
}

// Starts to copy 32 columns of 32 rows of an m x n array of 16-bit values (rows row0 ...,
// columns col0 ...) into the warp's shared memory, zeros for what is outside, four lanes
// a row.
template <typename T>
__device__ __forceinline__ void fetch_columns(unsigned char *to, const Matrix &in, int row0, int col0, int m, int n) {
    const int lane = threadIdx.x & 31, c = col0 + lane % 4 * 8;
    const bool whole = by_16<T>(in.p, in.stride) && c + 8 <= n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = row0 + i * 8 + lane / 4;
        const unsigned short *from = (const unsigned short *)in.p + (size_t)r * in.stride + c;
        unsigned char *place = to + (i * 8 + lane / 4) * 80 + lane % 4 * 16;
        if (c >= n || r >= m) {
            *(uint4 *)place = make_uint4(0, 0, 0, 0);
        } else if (whole) {
            copy_async(shared_address(place), from);
        } else {
            for (int j = 0; j < 8; ++j) ((unsigned short *)place)[j] = c + j < n ? from[j] : 0;
        }
    }
}
// This thread's row of them.
template <typename T>
__device__ __forceinline__ void get_columns(const unsigned char *from, float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Vec<T, 8> piece = load<T, 8>((const T *)(from + (threadIdx.x & 31) * 80) + 8 * j);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const Pair<float> two = piece.pair(q);
            v[8 * j + 2 * q] = two.x;
            v[8 * j + 2 * q + 1] = two.y;
        }
    }
}

// Which tile is worked on n-th: panels of `kPanel` tiles down, all columns of tiles
// across, so that the tiles in work at one time (one a multiprocessor) share rows
// of A and columns of B in L2.
constexpr int kPanel = 16;
struct Tile {
    int problem, split, row, column;
};
__device__ __forceinline__ Tile tile_of(int index, int down, int across, int splits) {
    Tile t;
    const int each = down * across, part = index / each;
    t.problem = part / splits;
    t.split = part - t.problem * splits;
    index -= part * each;
    const int panel = index / (kPanel * across), first = panel * kPanel;
    const int height = down - first < kPanel ? down - first : kPanel;
    index -= panel * kPanel * across;
    t.row = first + index % height;
    t.column = index / height;
    return t;
}

// TWICE: A comes as the sum of two arrays, each multiplied with the same tile of B. O: of what is written.
template <typename T, typename O, bool TWICE, int KIND, int BN, bool PAIR>
__global__ void __launch_bounds__(64 + 32 * epilogue_warps(KIND, TWICE), 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Product p, int down, int across, int tiles,
                   PipelineStarve starve) {
    constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kHidden || KIND == kInput || KIND == kWeights;
    constexpr int kWarps = epilogue_warps(KIND, TWICE);
    constexpr bool kInParts = TWICE || (KIND == kHidden && std::is_same_v<O, float>);  // of kChunk<T> blocks
    constexpr int kStages = stages_of(KIND, BN, TWICE, PAIR), kColumns = KIND == kGated ? BN / 2 : BN;  // of the result, a tile
    constexpr uint32_t kBytesA = bytes_a(TWICE), kStageBytes = stage_bytes(BN, TWICE, PAIR), kSumColumns = 2 * BN < 32 ? 32 : 2 * BN;
    extern __shared__ unsigned char memory[];
    __shared__ __align__(8) uint64_t barriers[2 * kStages + 5];
    __shared__ uint32_t sums_address;
    __shared__ volatile int gave_up;
    __shared__ uint32_t issued[2];   // blocks of K whose copies this block and (PAIR) the other one started, by rank
    __shared__ int other_gave_up;    // PAIR: a wait of the other block
    const uint32_t base = (shared_address(memory) + 1023) & ~1023u;
    unsigned char *staging = memory + (base - shared_address(memory)) + kStages * kStageBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Of the pair; tiles are taken by pairs.
    const int rank = PAIR ? (int)cooperative_groups::this_cluster().block_rank() : 0;
    const int team = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x, teams = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
    const uint32_t full = shared_address(barriers), empty = full + 8 * kStages, ready = empty + 8 * kStages,
                   taken = ready + 16, drained = taken + 16;
    if (threadIdx.x == 0) {
        gave_up = other_gave_up = 0;
        for (int s = 0; s < kStages; ++s) barrier_init(full + 8 * s, 1), barrier_init(empty + 8 * s, 1);
        for (int i = 0; i < 2; ++i) barrier_init(ready + 8 * i, 1), barrier_init(taken + 8 * i, (PAIR ? 2 : 1) * kWarps);
        barrier_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory is taken and given back by both blocks of a pair together, instructions
    // without a limit to their wait: the other block has to run when one asks, and may not
    // leave before both are through.
    if constexpr (PAIR) cooperative_groups::this_cluster().sync();
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             shared_address(&sums_address)),
                         "r"(kSumColumns)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             shared_address(&sums_address)),
                         "r"(kSumColumns)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    auto everyone = [&] {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if constexpr (PAIR) cooperative_groups::this_cluster().sync();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    everyone();
    const uint32_t sums = sums_address;
    const int blocks_k = (p.k + kBK - 1) / kBK;
    // A tile's blocks of K: all of them (kInput: once for each pair of operands), or its split's part.
    const int all = (KIND == kInput ? 2 : 1) * blocks_k;
    auto first_of = [&](const Tile &t) { return (int)((long long)all * t.split / p.splits); };
    auto last_of = [&](const Tile &t) { return (int)((long long)all * (t.split + 1) / p.splits); };
    after_previous();
    let_next_start();

    if (warp == 0 && lane == 0) {
        uint32_t step = 0;  // of all tiles, one after another
        // The box of A is no higher than A (its other rows are multiplied as they lie, for rows that do not exist).
        const uint32_t skipped = kAMn || PAIR ? 0 : kBytesA - box_rows(p.m) * kBK * 2;
        bool good = true;
        for (int index = team; index < tiles && good; index += teams) {
            const Tile t = tile_of(index, down, across, p.splits);
            const int last = last_of(t);
            for (int i = first_of(t); i < last; ++i, ++step) {
                const uint32_t s = step % kStages, round = step / kStages;
                if (step >= starve.block || !barrier_wait(empty + 8 * s, (round & 1) ^ 1, starve.polls, &gave_up)) {
                    good = false;
                    break;
                }
                const uint32_t to = base + s * kStageBytes;
                const uint32_t barrier = PAIR ? place_of(full + 8 * s, 0) : full + 8 * s;
                if (rank == 0) barrier_expect(full + 8 * s, (PAIR ? 2 : 1) * (kStageBytes - skipped));
                const int second = KIND == kInput && i >= blocks_k ? 1 : 0, k = (i - second * blocks_k) * kBK;
                const int row0 = (PAIR ? t.row * 2 + rank : t.row) * kBM;
                // This block's rows of B.
                constexpr int kHeld = PAIR ? BN / 2 : BN;
                const int col0 = t.column * (KIND == kGated ? kColumns : BN) + (KIND == kGated ? 0 : rank * kHeld);
                const CUtensorMap *a = &maps.a[KIND == kWeights ? t.problem : second];
                const CUtensorMap *b = &maps.b[KIND == kWeights ? t.problem : second];
                if constexpr (kAMn) {
                    for (int j = 0; j < kBM / 64; ++j) tma_load<PAIR>(to + j * 8192, a, row0 + j * 64, k, barrier);
                    if constexpr (TWICE)
                        for (int j = 0; j < kBM / 64; ++j)
                            tma_load<PAIR>(to + (kBM / 64 + j) * 8192, &maps.low[t.problem], row0 + j * 64, k, barrier);
                } else {
                    tma_load<PAIR>(to, a, k, row0, barrier);
                }
                if constexpr (kBMn) {
                    for (int j = 0; j < kHeld / 64; ++j)
                        tma_load<PAIR>(to + kBytesA + j * 8192, b, col0 + j * 64, k, barrier);
                } else if constexpr (KIND == kGated && PAIR) {  // gate's rows in one block, up's in the other
                    tma_load<PAIR>(to + kBytesA, &maps.b[rank], k, col0, barrier);
                } else if constexpr (KIND == kGated) {
                    tma_load<PAIR>(to + kBytesA, &maps.b[0], k, col0, barrier);
                    tma_load<PAIR>(to + kBytesA + bytes_b(kColumns), &maps.b[1], k, col0, barrier);
                } else {
                    tma_load<PAIR>(to + kBytesA, b, k, col0, barrier);
                }
            }
        }
        issued[rank] = step;
        if constexpr (PAIR) store_cluster(place_of(shared_address(&issued[rank]), rank ^ 1), step);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t kInstruction = instruction<T>(kAMn, kBMn, PAIR ? 2 * kBM : kBM, BN);
        uint32_t step = 0, round = 0;  // round: of the two places for sums
        bool good = true;
        for (int index = team; index < tiles && good; index += teams) {
            const Tile t = tile_of(index, down, across, p.splits);
            const int last = last_of(t);
            for (int i = first_of(t); i < last && good; ++round) {
                const uint32_t to = round & 1, use = round >> 1;
                const int first = i, end = kInParts && last - i > kChunk<T> ? i + kChunk<T> : last;
                good = barrier_wait(taken + 8 * to, (use & 1) ^ 1, starve.polls, &gave_up);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (; i < end && good; ++i, ++step) {
                    const uint32_t s = step % kStages;
                    if (!barrier_wait(full + 8 * s, (step / kStages) & 1, starve.polls, &gave_up)) {
                        good = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = base + s * kStageBytes;
                    const uint64_t a = operand(at, kAMn ? 8192 : 16), b = operand(at + kBytesA, kBMn ? 8192 : 16);
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k)  // 16 of K: 32 bytes along a row, or 16 rows of 128 bytes
                        multiply<PAIR>(sums + to * BN, a + (uint64_t)k * (kAMn ? 128 : 2), b + (uint64_t)k * (kBMn ? 128 : 2),
                                 kInstruction, i > first || k > 0);
                    if constexpr (TWICE) {
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)
                            multiply<PAIR>(sums + to * BN, a + (uint64_t)(bytes_a(false) / 16 + k * 128),
                                     b + (uint64_t)k * 128, kInstruction, true);
                    }
                    commit_to<PAIR>(empty + 8 * s);
                }
                if (good) commit_to<PAIR>(ready + 8 * to);
            }
        }
        // Matrix instructions in flight end before tensor memory is given back.
        commit_to<PAIR>(drained);
        barrier_wait(drained, 0, kPipelinePolls, nullptr);
    } else if (warp >= 2) {
        unsigned char *mine = staging + (warp - 2) * staging_of(KIND);
        const int quarter = warp & 3;  // the rows of tensor memory that this warp may read
        constexpr int kPart = kColumns / (kWarps / 4);  // its columns, from `begin` on
        const int begin = (warp - 2) / 4 * kPart;
        uint32_t round = 0;
        bool good = true;
        for (int index = team; index < tiles; index += teams) {
            const Tile t = tile_of(index, down, across, p.splits);
            const int row0 = (PAIR ? t.row * 2 + rank : t.row) * kBM + quarter * 32, row = row0 + lane;
            uint32_t at = 0;
            auto wait = [&] {  // for the next sums
                const uint32_t from = round & 1, use = round >> 1;
                if (good) good = barrier_wait(ready + 8 * from, use & 1, starve.polls, &gave_up);
                good = __all_sync(0xffffffffu, good);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                at = sums + from * BN + ((uint32_t)quarter << 21);
            };
            auto release = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                // A warp that gave up no longer says that it has taken what others may still be reading.
                if (lane == 0 && good) {
                    if constexpr (PAIR)
                        barrier_arrive_cluster(place_of(taken + 8 * (round & 1), 0));
                    else
                        barrier_arrive(taken + 8 * (round & 1));
                }
                ++round;
            };
            // What gave up is NaN from here on.
            auto take = [&](int c, float (&v)[32]) {
                if (good) {
                    take_columns(at + c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __int_as_float(0x7FC00000);
                }
            };
            // 32 columns of sum `which` of a part of K.
            auto put_partial = [&](const auto &v, int from, int which, int col0) {
                const size_t stride = partial_stride(p.n), part = (size_t)which * p.splits + t.split;
                put_columns<float>(mine, v, from, {(float *)p.partial + part * p.m * stride, stride}, row0, col0, p.m, p.n);
            };
            // float16's VJP: the powers of two of this tile's results.
            constexpr bool kTimes = std::is_same_v<T, __half> && (KIND == kHidden || KIND == kInput || KIND == kWeights);
            float times[3] = {1.0f, 1.0f, 1.0f};
            if constexpr (kTimes) {
#pragma unroll
                for (int n = 0; n < (KIND == kHidden ? 3 : 1); ++n) times[n] = times_of<T>(p, KIND == kWeights ? t.problem : n);
            }
            auto scale = [&](auto &v) {
                if constexpr (kTimes && KIND != kHidden) {
#pragma unroll
                    for (float &x : v) x *= times[0];
                }
            };
            // 32 columns of a result of kWeights, kDown, kInput.
            auto put = [&](const auto &v, int from, int col0) {
                if constexpr (KIND == kWeights) {
                    if (p.transposed[t.problem]) {
                        // A column of the tile is a row of the result: lanes are neighbours there.
                        const OutMatrix &out = p.out[t.problem];
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (row < p.m && col0 + j < p.n)
                                ((O *)out.p)[(size_t)(col0 + j) * out.stride + row] = narrow<O>(v[from + j]);
                        return;
                    }
                }
                put_columns<O>(mine, v, from, p.out[KIND == kWeights ? t.problem : 0], row0, col0, p.m, p.n);
            };
            // The sums of all parts of K but the last to be released, in registers.
            auto add_parts = [&](float (&sum)[kPart]) {
#pragma unroll
                for (int j = 0; j < kPart; ++j) sum[j] = 0.0f;
                const int last = last_of(t);
                for (int i = first_of(t); i < last; i += kChunk<T>) {
                    if (i > first_of(t)) release();
                    wait();
#pragma unroll
                    for (int c = 0; c < kPart; c += 32) {
                        float v[32];
                        take(begin + c, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[c + j] += v[j];
                    }
                }
            };
            if constexpr (TWICE) {
                float sum[kPart];
                add_parts(sum);
                release();
                if (p.splits == 1) scale(sum);
                if (row0 < p.m) {
#pragma unroll
                    for (int c = 0; c < kPart; c += 32) {
                        const int col0 = t.column * kColumns + begin + c;
                        if (col0 >= p.n) continue;
                        if (p.splits > 1)
                            put_partial(sum, c, t.problem, col0);
                        else
                            put(sum, c, col0);
                    }
                }
            } else {
                auto fetch = [&](int c) {
                    const int col0 = t.column * kColumns + c;
                    fetch_columns<T>(mine + 2 * kBox, p.saved[0], row0, col0, p.m, p.n);
                    fetch_columns<T>(mine + 2 * kBox + kRows, p.saved[1], row0, col0, p.m, p.n);
                    commit_async();
                };
                if constexpr (KIND == kHidden)
                    if (p.splits == 1) fetch(begin);
                if constexpr (kInParts) {
                    float sum[kPart];
                    add_parts(sum);
                    if (good) {  // to where the last part was, for what follows
#pragma unroll
                        for (int c = 0; c < kPart; c += 32) leave_columns(at + begin + c, sum + c);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                } else {
                    wait();
                }
                if (row0 < p.m) {
#pragma unroll 1
                    for (int c = begin; c < begin + kPart; c += 32) {
                        const int col0 = t.column * kColumns + c;
                        if (col0 >= p.n) break;
                        float v[32];
                        take(c, v);
                        if (p.splits > 1) {
                            put_partial(v, 0, KIND == kWeights ? t.problem : 0, col0);
                            if constexpr (KIND == kGated) {
                                take(kColumns + c, v);
                                put_partial(v, 0, 1, col0);
                            }
                            continue;
                        }
                        if constexpr (KIND == kGated) {
                            if (p.out[0].p != nullptr) put_columns<T>(mine, v, 0, p.out[0], row0, col0, p.m, p.n);
                            float u[32];
                            take(kColumns + c, u);
                            if (p.out[1].p != nullptr) put_columns<T>(mine, u, 0, p.out[1], row0, col0, p.m, p.n);
                            by_activation(p.activation, [&](auto kind) {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    v[j] = activation<true>(decltype(kind)::value, v[j], (float *)nullptr) * u[j];
                            });
                            put_columns<T>(mine, v, 0, p.out[2], row0, col0, p.m, p.n);
                        } else if constexpr (KIND == kHidden) {
                            // O float: with what the 16-bit values lose.
                            constexpr int kTerms = std::is_same_v<O, float> ? 2 : 1;
                            float g[32], u[32];
                            wait_async<0>();
                            __syncwarp();
                            get_columns<T>(mine + 2 * kBox, g);
                            get_columns<T>(mine + 2 * kBox + kRows, u);
                            __syncwarp();
                            if (c + 32 < begin + kPart) fetch(c + 32);  // on its way meanwhile
                            uint32_t words[3][kTerms][16];
                            by_activation(p.activation, [&](auto kind) {
#pragma unroll
                                for (int q = 0; q < 16; ++q) {
                                    Pair<float> f, slope;
                                    f.x = activation<true>(decltype(kind)::value, g[2 * q], &slope.x);
                                    f.y = activation<true>(decltype(kind)::value, g[2 * q + 1], &slope.y);
                                    const Pair<float> hb = {v[2 * q], v[2 * q + 1]}, up2 = {u[2 * q], u[2 * q + 1]};
                                    Pair<float> results[3] = {hb * up2 * slope, hb * f, f * up2};
                                    if constexpr (kTimes) {
#pragma unroll
                                        for (int n = 0; n < 3; ++n) results[n] = results[n] * both(times[n]);
                                    }
#pragma unroll
                                    for (int n = 0; n < 3; ++n) {
                                        words[n][0][q] = word_of<T>(results[n].x, results[n].y);
                                        if constexpr (kTerms == 2) {
                                            Vec<T, 2> high;
                                            high.w[0] = words[n][0][q];
                                            const Pair<float> left = results[n] + high.pair(0) * both(-1.0f);
                                            words[n][1][q] = word_of<T>(left.x, left.y);
                                        }
                                    }
                                }
                            });
                            int box = 0;
#pragma unroll
                            for (int n = 0; n < 3; ++n) {
                                if (p.out[n].p != nullptr)
                                    put_box(mine + (box++ & 1) * kBox, words[n][0], &maps.out[2 * n], row0, col0);
                                if constexpr (kTerms == 2)
                                    if (p.out_low[n].p != nullptr)
                                        put_box(mine + (box++ & 1) * kBox, words[n][1], &maps.out[2 * n + 1], row0, col0);
                            }
                            // The boxes in turn from chunk to chunk: an odd one out waits for both.
                            if (box & 1)
                                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        } else {
                            scale(v);
                            put(v, 0, col0);
                        }
                    }
                }
                release();
            }
        }
    }
    if constexpr (KIND == kHidden)
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    if constexpr (PAIR) {
        __syncthreads();
        if (threadIdx.x == 0 && gave_up) store_cluster(place_of(shared_address(&other_gave_up), rank ^ 1), 1);
    }
    everyone();
    if (PAIR && rank == 1 && threadIdx.x == 0)  // the first block's commits have arrived here too
        barrier_wait(drained, 0, kPipelinePolls, nullptr);
    if (gave_up || other_gave_up) {
        // Whichever wait it was: copies in flight land before a block ends. A stage's last copies were of the last round
        // begun; a pair's land at the first block's barriers, where one block may have come further than the other.
        if (threadIdx.x == 0 && rank == 0) {
            const uint32_t own = issued[0], other = PAIR ? issued[1] : own, most = own > other ? own : other;
            for (uint32_t n = most > (uint32_t)kStages ? most - kStages : 0; n < most; ++n) {
                const uint32_t barrier = full + 8 * (n % kStages);
                if (n >= own)
                    barrier_expect(barrier, kStageBytes);  // the other block's alone
                else if (n >= other)
                    barrier_excuse(barrier, kStageBytes);  // the other block's never began
                barrier_wait(barrier, (n / kStages) & 1, kPipelinePolls, nullptr);
            }
        }
    }
    __syncwarp();
    if (warp == 1) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(sums), "r"(kSumColumns) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sums), "r"(kSumColumns) : "memory");
    }
    if constexpr (PAIR) cooperative_groups::this_cluster().sync();
}

// ---- launches --------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// [rows][cols] in boxes of box_rows rows by 64 values (128 bytes, swizzled), or 32; zeros outside.
bool encode(CUtensorMap *map, bool bfloat, const Matrix &x, int rows, int cols, int box_rows, int box_cols = 64) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)x.stride * 2};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    const cuuint32_t each[2] = {1, 1};
    return map_encoder()(map, bfloat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void *>(x.p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename O, bool TWICE, int KIND, int BN, bool PAIR>
cudaError_t launch_tiles(const Product &p, PipelineStarve starve, cudaStream_t stream) {
    constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kHidden || KIND == kInput || KIND == kWeights;
    constexpr int kColumns = KIND == kGated ? BN / 2 : BN;
    constexpr bool kBfloat = std::is_same_v<T, __nv_bfloat16>;
    constexpr uint32_t kShared = shared_bytes(KIND, BN, TWICE, PAIR);
    constexpr int kThreads = 64 + 32 * epilogue_warps(KIND, TWICE);
    Maps maps = {};
    const int pairs_a = KIND == kInput ? 2 : p.problems, pairs_b = KIND == kInput || KIND == kGated ? 2 : p.problems;
    bool good = true;
    for (int i = 0; i < pairs_a; ++i) {
        good = good && (kAMn ? encode(&maps.a[i], kBfloat, p.a[i], p.k, p.m, kBK)
                             : encode(&maps.a[i], kBfloat, p.a[i], p.m, p.k, PAIR ? kBM : box_rows(p.m)));
        if (TWICE) good = good && encode(&maps.low[i], kBfloat, p.low[i], p.k, p.m, kBK);
    }
    for (int i = 0; i < pairs_b; ++i)
        good = good && (kBMn ? encode(&maps.b[i], kBfloat, p.b[i], p.k, p.n, kBK)
                             : encode(&maps.b[i], kBfloat, p.b[i], p.n, p.k, KIND == kGated || PAIR ? BN / 2 : BN));
    if constexpr (KIND == kHidden)
        for (int i = 0; i < 3; ++i) {
            if (p.out[i].p != nullptr)
                good = good && encode(&maps.out[2 * i], kBfloat, {p.out[i].p, p.out[i].stride}, p.m, p.n, 32, 32);
            if (p.out_low[i].p != nullptr)
                good = good && encode(&maps.out[2 * i + 1], kBfloat, {p.out_low[i].p, p.out_low[i].stride}, p.m, p.n, 32, 32);
        }
    if (!good) return cudaErrorInvalidValue;
    constexpr int kRowsAtOnce = PAIR ? 2 * kBM : kBM;
    const int down = (p.m + kRowsAtOnce - 1) / kRowsAtOnce, across = (p.n + kColumns - 1) / kColumns;
    const long long tiles = (long long)down * across * p.problems * p.splits;
    if (tiles > INT32_MAX) return cudaErrorInvalidValue;
    const auto kernel = product_kernel<T, O, TWICE, KIND, BN, PAIR>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared);
    if (e != cudaSuccess) return e;
    int most = geo::device_sm_count() / (PAIR ? 2 : 1);
    if constexpr (PAIR) {  // a pair needs two multiprocessors side by side
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)(2 * most));
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = kShared;
        cudaLaunchAttribute attribute = {};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = 2;
        attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        int resident = 0;
        e = cudaOccupancyMaxActiveClusters(&resident, kernel, &config);
        if (e != cudaSuccess) return e;
        if (resident > 0 && resident < most) most = resident;
    }
    return launch_after(kernel, (unsigned)((tiles < most ? tiles : most) * (PAIR ? 2 : 1)), kThreads, kShared,
                        PAIR ? 2 : 1, stream, maps, p, down, across, (int)tiles, starve);
}

template <typename T, typename O, bool TWICE, int KIND>
cudaError_t launch_kind(const Cut &cut, const Product &p, PipelineStarve starve, cudaStream_t stream) {
    if (cut.pair) return launch_tiles<T, O, TWICE, KIND, 256, true>(p, starve, stream);
    switch (cut.columns) {
        case 256: return launch_tiles<T, O, TWICE, KIND, 256, false>(p, starve, stream);
        case 128: return launch_tiles<T, O, TWICE, KIND, 128, false>(p, starve, stream);
        default: return launch_tiles<T, O, TWICE, KIND, 64, false>(p, starve, stream);
    }
}

template <typename T>
cudaError_t launch_type(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p, PipelineStarve starve,
                        cudaStream_t stream) {
    const bool to_float = out_type == GEO_B200_F32;
    const Cut cut = cut_tensor(kind, type, kind == kWeights && to_float, p.m, p.n, p.k);
    cudaError_t e;
    switch (kind) {
        case kGated: e = launch_kind<T, T, false, kGated>(cut, p, starve, stream); break;
        case kDown: e = launch_kind<T, T, false, kDown>(cut, p, starve, stream); break;
        case kHidden:
            e = to_float ? launch_kind<T, float, false, kHidden>(cut, p, starve, stream)
                         : launch_kind<T, T, false, kHidden>(cut, p, starve, stream);
            break;
        case kInput: e = launch_kind<T, T, false, kInput>(cut, p, starve, stream); break;
        default:
            e = to_float ? launch_kind<T, float, true, kWeights>(cut, p, starve, stream)
                         : launch_kind<T, T, false, kWeights>(cut, p, starve, stream);
            break;
    }
    return e != cudaSuccess || p.splits == 1 ? e : launch_join(kind, type, out_type, p, stream);
}

}  // namespace

bool tensor_products_available() { return map_encoder() != nullptr; }

// The cheapest by an estimate in cycles. A block of K costs what its matrix
// instructions take (4096 multiply-adds a cycle) or its copies (2 cycles and a bit for
// each row of 128 bytes: 600 cycles measured for 128 + 32 rows, 700 for 128 + 128, 670
// for a pair's 128 + 128), whichever is more; parts of K cost the way of their sums
// through L2 and one more launch.
Cut cut_tensor(ProductKind kind, uint32_t type, bool twice, size_t m, size_t n, size_t k) {
    const long long sms = geo::device_sm_count(), problems = kind == kWeights ? 3 : 1;
    const long long blocks = (long long)((k + kBK - 1) / kBK) * (kind == kInput ? 2 : 1);
    const long long rows_a = kind == kWeights ? kBM : box_rows((int)(m < (size_t)kBM ? m : kBM));
    const long long fewest = twice ? 1 : (blocks + longest(type) - 1) / longest(type);  // twice: summed up in registers
    Cut best = {256, false, (int)fewest};
    double least = -1;
    auto look = [&](int bn, bool pair) {
        const long long columns = kind == kGated ? bn / 2 : bn, high = pair ? 2 * kBM : kBM;
        const long long tiles = (long long)((m + high - 1) / high) * ((n + columns - 1) / columns) * problems;
        const long long teams = pair ? sms / 2 : sms, terms = twice ? 2 : 1;
        const double copies = 2.1 * (terms * rows_a + (pair ? bn / 2 : bn)) + 150, products = 2.0 * bn * terms;
        const double block = copies > products ? copies : products;
        for (long long splits = fewest; splits == fewest || (splits <= 16 && splits * 4 <= blocks); ++splits) {
            const long long waves = (tiles * splits + teams - 1) / teams;
            const double sums = (double)sums_of(kind, 3) * splits * m * n * 4;
            if (splits > fewest && (waves > 1 || sums > (64 << 20))) break;
            const double cost = waves * ((blocks + splits - 1) / splits * block + 800) + 4000 +
                                (splits > 1 ? 6500 + sums / 1800 : 0);
            if (least < 0 || cost < 0.98 * least) least = cost, best = {bn, pair, (int)splits};
        }
    };
    if (m > (size_t)kBM) look(256, true);
    for (int bn = 256; bn >= 64; bn /= 2) look(bn, false);
    return best;
}

cudaError_t launch_product_tensor(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p,
                                  PipelineStarve starve, cudaStream_t stream) {
    return type == GEO_B200_BF16 ? launch_type<__nv_bfloat16>(kind, type, out_type, p, starve, stream)
                                 : launch_type<__half>(kind, type, out_type, p, starve, stream);
}

}  // namespace layers
}  // namespace geo
