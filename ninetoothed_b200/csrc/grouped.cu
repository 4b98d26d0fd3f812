// Products whose weight matrix is chosen by the row: the rows of lhs form contiguous runs whose bounds lie on the
// device, and every run has its own matrix.
//
//   grouped_matmul           output[t] = lhs[t] . rhs[e]                       for the rows t of run e
//   grouped_matmul_rhs_grad  rhs_grad[e] = sum over the rows t of run e of lhs[t]^T output_grad[t]
//   lora_matmul              output[t] = lhs[t] . rhs + scales[a] (lhs[t] . down[a]) . up[a],  a the adapter of t's run
//
// Nothing is read back to the host: every CTA turns the offsets into a table of runs in shared memory (bounds are
// clamped by a running maximum, so no offsets can lead out of the tensors) and walks the tiles that follow from it.
//
// The kernels share a skeleton: persistent CTAs (or CTA pairs) of eleven warps or a few more, at least two that copy an operand
// each with TMA, one that issues tcgen05.mma, eight that drain the accumulator; a ring of shared-memory stages; two accumulator
// buffers in tensor memory, so that a tile's epilogue runs under the next tile's products.
//   turned_kernel   the grouped product (matrix columns are the accumulator's rows), the adapters' first product, and the
//                   whole of lora_matmul for few rows (with low_kernel before it)
//   lora_kernel     lora_matmul for many rows
//   grad_kernel     the gradient of the matrices
//   *_plain_kernel  operands that no tensor map can address
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "host.h"
#include "ptx.cuh"

namespace nt {
namespace {

constexpr int BM = 128;  // accumulator rows per CTA
constexpr int BK = 64;   // 64 16-bit elements: one 128-byte swizzle row
constexpr int UMMA_K = 16;
constexpr int A_STAGE_BYTES = BM * BK * 2;
constexpr int A_CHUNK_ROWS = 32;  // short tiles load only the 32-row boxes that hold rows of theirs
constexpr int TMEM_COLS = 512;
constexpr int MAX_STAGES = 8;
constexpr int MAX_RUNS = 2048;  // the table of runs is 16 bytes a run of shared memory
constexpr size_t MAX_SMEM = 227 * 1024;

// Warp 0 and the last copy, warp 1 issues the products, warps 2 to 9 are the epilogue (two a quadrant of the accumulator).
constexpr int EPILOGUE_WARPS = 8;
constexpr int ROW_WARP = 2 + EPILOGUE_WARPS;
constexpr int NUM_THREADS = (ROW_WARP + 1) * 32;
constexpr int ROW_PRODUCERS = 4;  // of lora_kernel
constexpr int SPLIT_WARP = ROW_WARP + ROW_PRODUCERS;
constexpr int SPLITTERS = 4;  // warps of lora_kernel that make fp16 adapters' operands from what the copies bring
constexpr int lora_threads(bool wide) { return (SPLIT_WARP + (wide ? SPLITTERS : 0)) * 32; }
constexpr int GRAD_THREADS = NUM_THREADS + 32;  // and a warp that clears what a run's last block holds of the next run

enum Job { JOB_PRODUCT, JOB_PARTS, JOB_FEW };  // of turned_kernel

constexpr int SPLIT_NT = 64;   // rows of a tile whose reduction a cluster shares
constexpr int FEW_RANK = 128;  // largest rank whose adapters' part may be computed a row at a time (see few_rows)
constexpr int LOW_WARPS = 8;
constexpr int LOW_CHUNK = LOW_WARPS * 256;  // terms of a partial sum of (lhs . down) there
constexpr int RANK_BLOCK = 32;  // ranks of one stage of the adapters' second product elsewhere: a 128-byte swizzle row of
                               // values, which are pairs of bf16 (32 first parts, 32 rests) or 32 bits wide

// A wait on a barrier tells a phase from the next one only, so no lane that goes through the ring of stages may fall a whole
// round behind: every producer has a part in `full`, by bytes that it copies into the stage or by arriving.
struct Control {
    uint64_t full[MAX_STAGES];
    uint64_t empty[MAX_STAGES];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t partials;
    uint64_t raw[MAX_STAGES];    // copies that warps of the CTA have to work on before products may read them
    uint64_t clean[MAX_STAGES];  // ... and that they have
    int tile_rows[MAX_STAGES];  // rows of the tiles whose stages are in the ring
    uint32_t tmem_base;
    uint32_t abort_flag;
    int runs;        // entries of the table
    int tiles_m;     // tile-rows of all runs
    int row_begin;   // rows covered by the offsets
    int row_end;
};

// One run of the table: rows [begin, end), the matrix it uses, the tile-rows of the runs before it.
struct Run {
    int begin, end, matrix, tiles_before;
};

constexpr int CONTROL_BYTES = 384;
static_assert(sizeof(Control) <= CONTROL_BYTES, "control block");

constexpr size_t table_bytes(int runs) { return static_cast<size_t>(runs + 1) * sizeof(Run); }

struct View {  // up to three dimensions; stride[0] is the matrix index's
    const void *data;
    int64_t stride[3];
};

struct Offsets {
    const void *data;
    int64_t stride;
    int wide;   // int64 elements, otherwise int32
    int runs;   // offsets holds runs + 1 bounds
};

struct Params {
    Offsets offsets;
    const void *adapters;  // matrix of every run (nullptr: run e uses matrix e)
    int64_t adapters_stride;
    int adapters_wide;
    int matrices;  // runs whose matrix lies outside 0 .. matrices - 1 have none
    int rows, n, k;
    int n_tiles, k_blocks, group_m;
    int bf16;
    void *out;
    int64_t out_stride0, out_stride1;
    int out_vec;  // rows of output are 16-byte addressable
    // adapters
    const float *scales;
    int64_t scales_stride;
    int rank, rank_blocks;
    int up_mn;  // up has unit stride along its columns, otherwise along its ranks
    int split;  // CTAs that share a tile's reduction
    // few rows under adapters: sums of (lhs . down) over chunks of the reduction [chunks, rows, rank], and up
    const float *low;
    int low_chunks;
    const void *up;
    int64_t up_stride[3];
    unsigned int *status;
};

__device__ __forceinline__ int load_index(const void *data, int64_t stride, int wide, int i, int low, int high) {
    const int64_t at = stride * i;
    const int64_t v = wide ? static_cast<const int64_t *>(data)[at] : static_cast<const int32_t *>(data)[at];
    return static_cast<int>(v < low ? low : v > high ? high : v);
}

// Fills the table with the runs that have rows (and, where adapters are given, an adapter, unless ALL: then runs without one
// have matrix -1), in row order.  All threads of the CTA call it; the table is complete after the next __syncthreads().
// Bounds outside 0 .. rows are clamped and a bound below an earlier one counts as that one, so that runs never overlap or
// leave the tensor.  tiles_before is in units of tiles, or with ALL in rows, of whole tiles all the same.
template <bool ALL>
__device__ __forceinline__ void build_table(const Params &p, Run *table, Control *ctl, int tile_m) {
    const int runs = p.offsets.runs;
    for (int i = threadIdx.x; i <= runs; i += blockDim.x) {
        table[i].begin = load_index(p.offsets.data, p.offsets.stride, p.offsets.wide, i, 0, p.rows);
        int matrix = i;
        if (p.adapters != nullptr && i < runs)
            matrix = load_index(p.adapters, p.adapters_stride, p.adapters_wide, i, -1, p.matrices);
        table[i].matrix = matrix;
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    const int first = table[0].begin;
    int bound = first, count = 0, tiles = 0;
    for (int base = 0; base < runs; base += 32) {
        const int i = base + lane;
        int end = i < runs ? table[i + 1].begin : 0;
        const int matrix = i < runs ? table[i].matrix : -1;
        __syncwarp();  // (entries are written below at places this chunk has read)
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end = max(end, other);
        }
        end = max(end, bound);
        int begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = bound;
        const bool valid = matrix >= 0 && matrix < p.matrices;
        const bool kept = i < runs && end > begin && (ALL || valid);
        const unsigned votes = __ballot_sync(0xffffffffu, kept);
        const int own_tiles = kept ? (end - begin + tile_m - 1) / tile_m : 0;
        int before = own_tiles;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += other;
        }
        if (kept) {
            // (at most entry `base + lane`; the bound of entry base + 32, still to be read as a next bound's
            // predecessor, is carried in `bound`)
            table[count + __popc(votes & ((1u << lane) - 1))] =
                Run{begin, end, valid ? matrix : -1, (tiles + before - own_tiles) * (ALL ? tile_m : 1)};
        }
        count += __popc(votes);
        tiles += __shfl_sync(0xffffffffu, before, 31);
        bound = __shfl_sync(0xffffffffu, end, 31);
        __syncwarp();
    }
    if (lane == 0) {
        ctl->runs = count;
        ctl->tiles_m = tiles;
        ctl->row_begin = first;
        ctl->row_end = bound;
    }
}

// The run that holds `row`, or -1: the one before the first bound above it (a bound above `row` that comes first ends
// the run by the running maximum too).  A warp looks at 256 bounds at a time, for one memory latency.
__device__ __forceinline__ int run_of(const Offsets &o, int rows, int row) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base <= o.runs; base += 256) {
        bool above[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = base + j * 32 + lane;
            above[j] = i <= o.runs && load_index(o.data, o.stride, o.wide, i, 0, rows) > row;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned votes = __ballot_sync(0xffffffffu, above[j]);
            if (votes != 0) return base + j * 32 + __ffs(votes) - 2;
        }
    }
    return -1;
}

// The adapter of `row`, or -1 (whole warps call it).
__device__ __forceinline__ int adapter_of(const Params &p, int row) {
    const int run = run_of(p.offsets, p.rows, row);
    if (run < 0) return -1;
    const int adapter = load_index(p.adapters, p.adapters_stride, p.adapters_wide, run, -1, p.matrices);
    return adapter < p.matrices ? adapter : -1;
}

// The rows covered by all runs: from the first bound to the largest.
__device__ __forceinline__ void build_range(const Params &p, Control *ctl) {
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int largest = 0;
    for (int i = lane; i <= p.offsets.runs; i += 32)
        largest = max(largest, load_index(p.offsets.data, p.offsets.stride, p.offsets.wide, i, 0, p.rows));
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (lane == 0) {
        ctl->row_begin = load_index(p.offsets.data, p.offsets.stride, p.offsets.wide, 0, 0, p.rows);
        ctl->row_end = largest;
        ctl->tiles_m = (largest - ctl->row_begin + SPLIT_NT - 1) / SPLIT_NT;
        ctl->runs = 0;
    }
}

__device__ __forceinline__ void raster(int tile, int m_tiles, int n_tiles, int group_m, int &m, int &n) {
    if (m_tiles <= group_m) {  // one group: a division is some 100 cycles between two tiles
        n = m_tiles == 1 ? tile : tile / m_tiles;
        m = tile - n * m_tiles;
        return;
    }
    const int per_group = group_m * n_tiles;
    const int group = tile / per_group;
    const int first = group * group_m;
    const int height = min(m_tiles - first, group_m);
    const int inside = tile - group * per_group;
    m = first + inside % height;
    n = inside / height;
    if (group & 1) n = n_tiles - 1 - n;  // odd groups walk back, starting on the panels the previous one ended on
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
    uint32_t packed;
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        packed = *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        packed = *reinterpret_cast<const uint32_t *>(&v);
    }
    return packed;
}

// A value as the sum of two numbers, its first `bits` bits and the rest (which the caller rounds), for a second product with each.
// Where an element of up is infinite both products have to be infinite with the value's sign, so neither part is zero or of the
// other sign: the first bits are cut off, not rounded, and a value that has no others is halved.  (Of values below 2^-100 the
// second part may still be zero.)  Both parts of an infinity or NaN are the value.
struct TwoParts {
    float first, rest;
    __device__ TwoParts(float v, int bits) {
        first = __uint_as_float(__float_as_uint(v) & (0xffffffffu << (24 - bits)));
        rest = v - first;
        if (rest == 0.f) first = rest = 0.5f * v;
        if (!isfinite(v)) first = rest = v;
    }
};

__device__ __forceinline__ void store16(void *out, int64_t at, float v, bool bf16) {
    if (bf16) static_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half *>(out)[at] = __float2half_rn(v);
}

__device__ __forceinline__ float load16(const void *in, int64_t at, bool bf16) {
    return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(in)[at])
                : __half2float(static_cast<const __half *>(in)[at]);
}

// A copy costs a lone lane about 130 cycles to issue, so the operands have a producer each and stages are 128 deep where they
// can be: a stage's copies take less than its products.
template <int CG>
__device__ __forceinline__ void load_2d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y) {
    if constexpr (CG == 1) tma_load_2d(dst, map, bar, x, y);
    else tma_load_2d_pair(dst, map, bar, x, y);
}

template <int CG>
__device__ __forceinline__ void load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z) {
    if constexpr (CG == 1) tma_load_3d(dst, map, bar, x, y, z);
    else tma_load_3d_pair(dst, map, bar, x, y, z);
}

// ---------------------------------------------------------------------------
// The grouped product with its operands' parts exchanged: 128 columns of a run's matrix (256 on a CTA pair) are the
// rows of the accumulator and up to NT of the run's rows its columns, so that a tile's width follows the number of
// rows it has, in steps of 16 (32), and no part of an instruction is spent on rows of nobody.
//
// SPLIT: a cluster of CTAs shares a tile, each taking a share of the reduction, for calls with fewer tiles than the
// device has SMs.  Every CTA adds up and stores the tile's rows of one share, reading the others' partial sums, in
// the order of the CTAs, from its own shared memory, where they have put them.
//
// What bounds it: for short runs the matrices, each read once: 64 of 2048 x 1024 for 256 rows take 45.6 us, 5.5 TB/s; the two
// 4096 x 2048 matrices of two single rows 11 us, of which 5 are their bytes and the rest a launch, a table and the first
// copy's latency.  For long runs the products and the board's power: 16384 rows over 16 matrices of 2048 x 4096 take 206 us in a
// short burst, with the tensor pipe at work 79 % of the time, 246 (1.1 PFLOP/s) back to back; 16 equal dense products of the same
// size as a library's batch 225.  In between nothing is near its limit: 64 runs of 256 rows on average against 2048 x 1024
// matrices take 98 us, with the tensor pipe at work 42 % of the time, 4 TB/s of DRAM, and 33 bytes a cycle into an SM, which
// takes in 64; 29 runs of 172 rows against 1544 x 1160 ones 41 us, with 24 %, 2.6 TB/s and 20 bytes.
// ---------------------------------------------------------------------------
template <int CG, int NT>
struct Turned {
    static constexpr int ROWS_CTA = NT / CG;  // rows of lhs that a CTA loads at most
    // Stages are two 64-deep blocks: half the barriers, and one box holds 128 rows of a matrix.  (A 64-deep block cost its
    // producer and its issuer 440 cycles whatever its width, more than the products of a narrow tile take.)
    static constexpr int SUB = 2;
    static constexpr int DEPTH = BK * SUB;
    static constexpr int W_BYTES = A_STAGE_BYTES * SUB;
    static constexpr int X_BYTES = ROWS_CTA * BK * 2;  // one 64-deep block of them
    static constexpr int STAGE_BYTES = W_BYTES + X_BYTES * SUB;
    static constexpr int STAGES = 192 * 1024 / STAGE_BYTES < MAX_STAGES ? 192 * 1024 / STAGE_BYTES : MAX_STAGES;
    static constexpr int TILE_N = BM * CG;
};
constexpr int SPLIT_STAGES = 3;
constexpr int SPLIT_BYTES = SPLIT_NT * BM * 4;  // partial sums: for every CTA of the cluster, its share of the rows

template <int CG, int NT, bool SPLIT>
constexpr int turned_stages() {
    return SPLIT ? SPLIT_STAGES : Turned<CG, NT>::STAGES;
}

constexpr int FEW_BYTES = SPLIT_NT * FEW_RANK * 4;  // (lhs . down) of a CTA's rows

template <int CG, int NT, bool SPLIT, bool FEW>
constexpr size_t turned_smem(int runs) {
    return 1024 + turned_stages<CG, NT, SPLIT>() * Turned<CG, NT>::STAGE_BYTES + CONTROL_BYTES + (SPLIT ? SPLIT_BYTES : 0) +
           (FEW ? FEW_BYTES : table_bytes(runs));
}

// A tile: rows [row0, row0 + rows) of a run against columns from col0 of its matrix.
struct TurnedPlace {
    int row0, rows, col0, matrix;
};

template <int CG, int NT, bool FEW>
struct TurnedWalk {
    const Run *table;
    int tile, total, stride, runs, run, range_begin, range_end;

    __device__ TurnedWalk(const Params &p, const Run *table_, const Control *ctl, int first, int step)
        : table(table_), tile(first), total(ctl->tiles_m * p.n_tiles), stride(step), runs(ctl->runs), run(0),
          range_begin(ctl->row_begin), range_end(ctl->row_end) {
        int high = FEW ? 0 : runs - 1;
        while (run < high) {  // the last run whose first tile is not behind this one
            const int mid = (run + high + 1) >> 1;
            if (table[mid].tiles_before * p.n_tiles <= tile) run = mid;
            else high = mid - 1;
        }
    }
    __device__ bool more() const { return tile < total; }
    __device__ void advance() { tile += stride; }
    __device__ TurnedPlace place(const Params &p) {
        if constexpr (FEW) {  // all rows against one matrix
            const int n = tile % p.n_tiles, first = range_begin + tile / p.n_tiles * NT;
            return {first, min(NT, range_end - first), n * Turned<CG, NT>::TILE_N, 0};
        } else {
            while (run + 1 < runs && table[run + 1].tiles_before * p.n_tiles <= tile) ++run;
            const Run r = table[run];
            const int length = r.end - r.begin, tiles = (length + NT - 1) / NT;
            constexpr int STEP = 16 * CG;
            const int even = tiles == 1 ? length : (length + tiles - 1) / tiles;
            const int share = (even + STEP - 1) / STEP * STEP;  // rows of a tile, in whole steps
            int m, n;
            raster(tile - r.tiles_before * p.n_tiles, tiles, p.n_tiles, p.group_m, m, n);
            return {r.begin + m * share, min(share, length - m * share), n * Turned<CG, NT>::TILE_N, r.matrix};
        }
    }
};

// The address of this CTA's shared-memory location in another CTA of the cluster, and a store to such an address.
__device__ __forceinline__ uint32_t remote_address(const void *local, uint32_t cta) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(cta));
    return remote;
}
__device__ __forceinline__ void store_remote(uint32_t address, const float4 &v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(address), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Partial sums lie four rows together: element (row r, column n) of a CTA's part is float r % 4 of float4 r / 4 * 128 + n.
// The rows that each CTA of the cluster adds up and stores, a whole number of fours.
__device__ __forceinline__ int split_share(int rows, int split) { return ((rows + split - 1) / split + 3) / 4 * 4; }

// Bounded wait for arrivals that come from other CTAs of the cluster with data they have written here.
__device__ __forceinline__ void mbar_wait_cluster(uint64_t *bar, uint32_t parity, const WaitCtx &ctx, uint32_t code) {
    for (int i = 0; i < 256; ++i)
        if (mbar_test_wait_cluster(bar, parity)) return;
    const uint64_t start = global_timer_ns();
    while (!mbar_test_wait_cluster(bar, parity)) {
        const bool failed_before = *ctx.abort_flag != 0;
        if (global_timer_ns() - start > (failed_before ? WAIT_LIMIT_AFTER_FAILURE_NS : WAIT_LIMIT_NS)) {
            if (!failed_before) {
                *ctx.abort_flag = 1;
                atomicCAS(ctx.status, 0u, STATUS_WAIT_TIMEOUT | (ctx.kernel_id << 16) | code);
            }
            return;
        }
    }
}

// Bounded wait of a warp that issues products, by all of it together: one lane probes, the warp's vote says whether to go on.
// (32 lanes probing one barrier are served one after the other.)
template <bool CLUSTER = false>
__device__ __forceinline__ void mbar_wait_together(uint64_t *bar, uint32_t parity, const WaitCtx &ctx, uint32_t code) {
    const bool prober = (threadIdx.x & 31) == 0;
    uint64_t start = 0;
    for (uint32_t i = 0;; ++i) {
        bool over = true;
        if (prober) over = CLUSTER ? mbar_test_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
        if (__all_sync(0xffffffffu, over)) break;
        if (i < 64 || i % 32 != 0) continue;
        if (prober) {
            const uint64_t now = global_timer_ns();
            if (start == 0) start = now;
            const bool failed_before = *ctx.abort_flag != 0;
            over = now - start > (failed_before ? WAIT_LIMIT_AFTER_FAILURE_NS : WAIT_LIMIT_NS);
            if (over && !failed_before) {
                *ctx.abort_flag = 1;
                atomicCAS(ctx.status, 0u, STATUS_WAIT_TIMEOUT | (ctx.kernel_id << 16) | code);
            }
        }
        if (__all_sync(0xffffffffu, over)) break;
    }
    __syncwarp();
}

// An arrival at the even CTA's barrier that tells of no writes.  (As a release it would have this lane wait for its copies' issue.)
__device__ __forceinline__ void arrive_leader(uint64_t *bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_address(bar, 0)) : "memory");
}

__device__ __forceinline__ void griddepcontrol_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddepcontrol_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async;" ::: "memory"); }

__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(EPILOGUE_WARPS * 32) : "memory"); }

__device__ __forceinline__ float half_of(uint32_t pair, int i, bool bf16) {
    const uint32_t bits = i ? pair >> 16 : pair & 0xffffu;
    return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// 16 bytes or less of a row of 16-bit values from `at` on, zeros behind `left` elements.  Aligned to `N` elements.
template <int N>
__device__ __forceinline__ void load_values(const uint16_t *at, int left, bool bf16, float (&v)[N]) {
    if (left >= N) {
        uint32_t words[N / 2];
        if constexpr (N == 8) *reinterpret_cast<uint4 *>(words) = __ldg(reinterpret_cast<const uint4 *>(at));
        else *reinterpret_cast<uint2 *>(words) = __ldg(reinterpret_cast<const uint2 *>(at));
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = half_of(words[j / 2], j & 1, bf16);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < left ? load16(at, j, bf16) : 0.f;
    }
}

__device__ __forceinline__ void prefetch_l2(const void *at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }

// Sixteen ranks of four columns of up, from rank r0 on: eight bytes a rank where a rank's columns lie side by side, two times
// sixteen bytes a column where a column's ranks do (their number is a multiple of eight then).  Ranks behind the last are 0.
__device__ __forceinline__ void load_ranks(const Params &p, const uint16_t *matrix, int col, int r0, uint32_t (&v)[32]) {
    if (p.up_mn) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint2 w = r0 + r < p.rank ? __ldg(reinterpret_cast<const uint2 *>(matrix + (r0 + r) * p.up_stride[1] + col)) : make_uint2(0, 0);
            v[2 * r] = w.x;
            v[2 * r + 1] = w.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + i % 2 * 8;
            const uint4 w = r < p.rank ? __ldg(reinterpret_cast<const uint4 *>(matrix + (col + i / 2) * p.up_stride[2] + r)) : make_uint4(0, 0, 0, 0);
            v[4 * i] = w.x;
            v[4 * i + 1] = w.y;
            v[4 * i + 2] = w.z;
            v[4 * i + 3] = w.w;
        }
    }
}

// ... times the row's (lhs . down).
__device__ __forceinline__ void add_ranks(const Params &p, const uint32_t (&v)[32], const float *l, int r0, bool bf16, float (&sum)[4]) {
    if (p.up_mn) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float weight = r0 + r < p.rank ? l[r0 + r] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] = fmaf(weight, half_of(v[2 * r + j / 2], j & 1, bf16), sum[j]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float weight = r0 + r < p.rank ? l[r0 + r] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] = fmaf(weight, half_of(v[8 * j + r / 2], r & 1, bf16), sum[j]);
        }
    }
}

// scales (lhs . down) . up of the rows that this CTA stores into its own slot of the partial sums.  A warp takes every
// eighth row, a lane four columns of the tile.  It is all memory latency, and a load waits behind the copies that stream the
// tile's operands: a step is done for all of the warp's rows at once, and what does not depend on the launch before (which
// adapter, its matrix on the way to L2, its first ranks for the first two rows in registers) before the wait for it.
__device__ __forceinline__ void adapters_part(const Params &p, const TurnedPlace &at, float *partials, float *low, int cta_rank,
                                              int split) {
    const int warp = static_cast<int>(threadIdx.x) / 32 - 2, lane = threadIdx.x & 31;
    const bool bf16 = p.bf16 != 0;
    const int share = split_share(at.rows, split);
    const int first = cta_rank * share, mine = min(at.rows, first + share) - first;
    const int row0 = at.row0 + first, col = at.col0 + lane * 4, left = p.n - col;
    const int rows = mine > warp ? (mine - warp + EPILOGUE_WARPS - 1) / EPILOGUE_WARPS : 0;  // of this warp, at most eight
    const uint16_t *up = static_cast<const uint16_t *>(p.up);
    // lane i looks after the warp's i-th row, row0 + warp + 8 i
    int run = -1, open = rows > 0 ? (1 << rows) - 1 : 0;  // rows whose run is not found yet
    for (int base = 0; base <= p.offsets.runs && open != 0; base += 256) {
        int bound[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = base + j * 32 + lane;
            bound[j] = i <= p.offsets.runs ? load_index(p.offsets.data, p.offsets.stride, p.offsets.wide, i, 0, p.rows) : INT_MIN;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (base + j * 32 > p.offsets.runs || open == 0) break;
            for (int i = 0; i < rows; ++i) {
                if (!(open >> i & 1)) continue;
                const unsigned votes = __ballot_sync(0xffffffffu, bound[j] > row0 + warp + EPILOGUE_WARPS * i);
                if (votes == 0) continue;
                open &= ~(1 << i);  // (the run before the first bound above the row: see run_of)
                if (lane == i) run = base + j * 32 + __ffs(votes) - 2;
            }
        }
    }
    int adapter = -1;
    float scale = 0.f;
    if (lane < rows && run >= 0) {
        adapter = load_index(p.adapters, p.adapters_stride, p.adapters_wide, run, -1, p.matrices);
        if (adapter >= p.matrices) adapter = -1;
        if (adapter >= 0) scale = p.scales[adapter * p.scales_stride];
    }
    for (int i = 0; i < rows; ++i) {
        const int which = __shfl_sync(0xffffffffu, adapter, i);
        if (which < 0) continue;
        const uint16_t *matrix = up + which * p.up_stride[0];
        if (p.up_mn) {
            for (int q = lane; q < 2 * p.rank; q += 32)
                if (at.col0 + (q & 1) * 64 < p.n) prefetch_l2(matrix + (q / 2) * p.up_stride[1] + at.col0 + (q & 1) * 64);
        } else {
            for (int j = 0; j < 4 && j < left; ++j)
                for (int r = 0; r < p.rank; r += 64) prefetch_l2(matrix + (col + j) * p.up_stride[2] + r);
        }
    }
    const bool wide = left >= 4 && (p.up_mn || p.rank % 8 == 0);  // this lane's columns come in whole loads
    const auto matrix_of = [&](int i) {
        const int which = __shfl_sync(0xffffffffu, adapter, i);
        return which < 0 || i >= rows ? nullptr : up + which * p.up_stride[0];
    };
    const uint16_t *m0 = matrix_of(0), *m1 = matrix_of(1);
    uint32_t v0[32], v1[32];
    if (wide && m0 != nullptr) load_ranks(p, m0, col, 0, v0);
    if (wide && m1 != nullptr) load_ranks(p, m1, col, 0, v1);
    griddepcontrol_wait();  // (the sums of lhs . down come from the launch before)
#pragma unroll 4
    for (int q = lane; q < rows * p.rank; q += 32) {
        const int i = q / p.rank, t = warp + EPILOGUE_WARPS * i;
        const float *part = p.low + static_cast<int64_t>(row0 + t) * p.rank + (q - i * p.rank);
        float total = 0.f;
        for (int c = 0; c < p.low_chunks; ++c) total += __ldcg(part + static_cast<int64_t>(c) * p.rows * p.rank);
        low[t * p.rank + (q - i * p.rank)] = total;
    }
    __syncwarp();
    for (int i = 0; i < rows; i += 2) {
        const int t0 = warp + EPILOGUE_WARPS * i, t1 = t0 + EPILOGUE_WARPS;
        const float *l0 = low + t0 * p.rank, *l1 = low + t1 * p.rank;
        if (i > 0) {
            m0 = matrix_of(i);
            m1 = matrix_of(min(i + 1, 31));
        }
        float sum0[4] = {}, sum1[4] = {};
        if (wide) {
            for (int r0 = 0; r0 < p.rank; r0 += 16) {
                if (i > 0 || r0 > 0) {
                    if (m0 != nullptr) load_ranks(p, m0, col, r0, v0);
                    if (m1 != nullptr) load_ranks(p, m1, col, r0, v1);
                }
                if (m0 != nullptr) add_ranks(p, v0, l0, r0, bf16, sum0);
                if (m1 != nullptr) add_ranks(p, v1, l1, r0, bf16, sum1);
            }
        } else {
            for (int r = 0; r < p.rank; ++r)
                for (int j = 0; j < 4 && j < left; ++j) {
                    const int64_t at_up = r * p.up_stride[1] + (col + j) * p.up_stride[2];
                    if (m0 != nullptr) sum0[j] = fmaf(l0[r], load16(m0, at_up, bf16), sum0[j]);
                    if (m1 != nullptr) sum1[j] = fmaf(l1[r], load16(m1, at_up, bf16), sum1[j]);
                }
        }
        const float s0 = __shfl_sync(0xffffffffu, scale, i), s1 = __shfl_sync(0xffffffffu, scale, i + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            partials[((cta_rank * share + t0) / 4 * BM + lane * 4 + j) * 4 + t0 % 4] = m0 != nullptr ? s0 * sum0[j] : 0.f;
            if (i + 1 < rows)
                partials[((cta_rank * share + t1) / 4 * BM + lane * 4 + j) * 4 + t1 % 4] = m1 != nullptr ? s1 * sum1[j] : 0.f;
        }
    }
    epilogue_sync();
}

// Partial sums of lhs . down over chunks of the reduction, for calls with few rows: a block takes a row, a chunk and eight
// ranks, a warp 256 terms of them.  All latency: every lane's loads are independent, and its part of the row is asked for
// before the row's adapter is looked up.  (One row, 4096 x 4096, rank 16: 14 us with the projection that starts under it, whose
// matrix alone takes 5; 64 rows of 64 requests 22.5.)
__global__ void __launch_bounds__(LOW_WARPS * 32) low_kernel(const __grid_constant__ Params p, const void *lhs, int64_t lhs_stride0,
                                                             View down, int down_mn, float *low) {
    griddepcontrol_launch_dependents();  // (the projection starts at once and waits for this kernel before it reads `low`)
    __shared__ float sums[LOW_WARPS][8];
    const bool bf16 = p.bf16 != 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, groups = (p.rank + 7) / 8;
    const int task = blockIdx.x, row = task / (p.low_chunks * groups), rest = task - row * (p.low_chunks * groups);
    const int chunk = rest / groups, r0 = (rest - chunk * groups) * 8;
    const int k0 = chunk * LOW_CHUNK + warp * 256;
    const uint16_t *x = static_cast<const uint16_t *>(lhs) + row * lhs_stride0;
    float xs[8];
    if (down_mn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) xs[i] = k0 + i * 32 + lane < p.k ? load16(x, k0 + i * 32 + lane, bf16) : 0.f;
    } else {
        load_values<8>(x + k0 + lane * 8, p.k - (k0 + lane * 8), bf16, xs);
    }
    const int adapter = adapter_of(p, row);
    if (adapter < 0) return;
    const uint16_t *d = static_cast<const uint16_t *>(down.data) + adapter * down.stride[0];
    float acc[8] = {};
    if (down_mn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = k0 + i * 32 + lane;
            if (k >= p.k) continue;
            float v[8];
            load_values<8>(d + k * down.stride[1] + r0, p.rank - r0, bf16, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(xs[i], v[j], acc[j]);
        }
    } else {
        const int k = k0 + lane * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (r0 + j >= p.rank || k >= p.k) continue;
            float v[8];
            load_values<8>(d + (r0 + j) * down.stride[2] + k, p.k - k, bf16, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[j] = fmaf(xs[i], v[i], acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int d2 = 16; d2 > 0; d2 /= 2) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], d2);
    float mine = acc[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mine = lane == j ? acc[j] : mine;
    if (lane < 8) sums[warp][lane] = mine;
    __syncthreads();
    if (threadIdx.x < 8 && r0 + static_cast<int>(threadIdx.x) < p.rank) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < LOW_WARPS; ++w) sum += sums[w][threadIdx.x];
        low[(static_cast<int64_t>(chunk) * p.rows + row) * p.rank + r0 + threadIdx.x] = sum;
    }
}

// 32 rows of a turned accumulator: lane l holds column n of all of them and the warp's 32 columns are neighbours.  Three
// exchanges with the lanes 1, 2 and 4 away leave every lane with eight neighbouring columns of every eighth row, which
// are 16-byte stores.  (One 2-byte store a row and lane took 80 cycles a row: more than the products of 2048 terms.)
// The first sixteen columns of the accumulator are rows from row0 on, `rows0` of them, the others from row1 on.
__device__ __forceinline__ void store_turned(const uint32_t (&acc)[32], void *out, int64_t stride0, int64_t row0, int rows0,
                                             int64_t row1, int rows1, int n, int n_end, bool bf16) {
    const int lane = threadIdx.x & 31;
    const bool odd1 = lane & 1, odd2 = lane & 2, odd4 = lane & 4;
    uint32_t pair[16];  // two columns of row 2i + (lane & 1)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd1 ? acc[2 * i] : acc[2 * i + 1], 1);
        pair[i] = pack2(__uint_as_float(odd1 ? other : acc[2 * i]), __uint_as_float(odd1 ? acc[2 * i + 1] : other), bf16);
    }
    uint32_t four[8][2];  // four columns of row 4i + (lane & 3)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, odd2 ? pair[2 * i] : pair[2 * i + 1], 2);
        four[i][0] = odd2 ? other : pair[2 * i];
        four[i][1] = odd2 ? pair[2 * i + 1] : other;
    }
    const int col = n - (lane & 7);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // eight columns of row 8i + (lane & 7)
        const uint32_t other0 = __shfl_xor_sync(0xffffffffu, odd4 ? four[2 * i][0] : four[2 * i + 1][0], 4);
        const uint32_t other1 = __shfl_xor_sync(0xffffffffu, odd4 ? four[2 * i][1] : four[2 * i + 1][1], 4);
        uint4 v;
        v.x = odd4 ? other0 : four[2 * i][0];
        v.y = odd4 ? other1 : four[2 * i][1];
        v.z = odd4 ? four[2 * i + 1][0] : other0;
        v.w = odd4 ? four[2 * i + 1][1] : other1;
        const int row = 8 * (i & 1) + (lane & 7);
        if (row < (i < 2 ? rows0 : rows1) && col < n_end) {
            uint16_t *dst = static_cast<uint16_t *>(out) + ((i < 2 ? row0 : row1) + row) * stride0 + col;
            if (col + 8 <= n_end) {
                *reinterpret_cast<uint4 *>(dst) = v;
            } else {
                const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (col + j < n_end) dst[j] = static_cast<uint16_t>(words[j / 2] >> (16 * (j & 1)));
            }
        }
    }
}

// JOB_PARTS: a run's adapter's down is the matrix, and scales (lhs . down) leaves in blocks of 32 ranks, 32 bits a rank: of fp16
// operands as it is, of bf16 ones as 32 first parts and 32 rests (their sum is the value to 2^-16, so that the second product runs
// on the tensor cores without the rounding of one 16-bit operand; bf16 has the range of fp32, fp16 has not).  Ranks behind the
// last are zero (of an infinite row or scale too).
// JOB_FEW: the shared projection and the adapters of a call with few rows.  The epilogue's warps, idle while the tile's
// products run, compute the adapters' part of the rows that their CTA will store, (lhs . down) . up in fp32, and put it
// where the CTA's own partial sums are added to it.
template <int CG, int NT, bool W_MN, bool SPLIT, Job JOB>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    turned_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ CUtensorMap map_x_chunk, const __grid_constant__ Params p) {
    using S = Turned<CG, NT>;
    constexpr bool FEW = JOB == JOB_FEW, PARTS = JOB == JOB_PARTS;
    constexpr int STAGES = turned_stages<CG, NT, SPLIT>();
    static_assert(!SPLIT || (CG == 1 && NT == SPLIT_NT), "a cluster that splits the reduction holds single CTAs");
    static_assert(!FEW || SPLIT, "few rows");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Control *ctl = reinterpret_cast<Control *>(smem + STAGES * S::STAGE_BYTES);
    float *partials = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(ctl) + CONTROL_BYTES);
    // (one or the other)
    Run *table = reinterpret_cast<Run *>(reinterpret_cast<uint8_t *>(partials) + (SPLIT ? SPLIT_BYTES : 0));
    float *low = reinterpret_cast<float *>(table);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const WaitCtx wait_ctx{&ctl->abort_flag, p.status, KID_GROUPED};
    const uint32_t cta_rank = CG == 1 && !SPLIT ? 0u : cluster_cta_rank();
    const bool leader = SPLIT || cta_rank == 0;
    const int split = SPLIT ? p.split : 1;
    const int worker = blockIdx.x / (SPLIT ? split : CG), workers = gridDim.x / (SPLIT ? split : CG);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], EPILOGUE_WARPS * 32 * CG);
        }
        if constexpr (SPLIT) mbar_init(&ctl->partials, EPILOGUE_WARPS * split);
        ctl->abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_x_chunk);
    }
    if (warp == 1) {
        tmem_alloc<CG>(&ctl->tmem_base, TMEM_COLS);
        tmem_relinquish<CG>();
    }
    if constexpr (FEW) build_range(p, ctl);
    else build_table<false>(p, table, ctl, NT);
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if constexpr (SPLIT) cluster_arrive();  // (awaited before the first access to another CTA's memory)
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    if constexpr (PARTS) griddepcontrol_launch_dependents();  // (the projection waits for this kernel before it reads the parts)
    using W = TurnedWalk<CG, NT, FEW>;
    // this CTA's share of the reduction (a share may be empty)
    const int kb_first = SPLIT ? p.k_blocks * static_cast<int>(cta_rank) / split : 0;
    const int kb_last = SPLIT ? p.k_blocks * (static_cast<int>(cta_rank) + 1) / split : p.k_blocks;

    if (warp == 0 || warp == ROW_WARP) {
        // ------------- TMA producers: warp 0 the matrices, the last warp the rows -------------
        // (Lone lanes, in branches that no other lane of the warp enters: these loops go by values from shared memory, and in a
        // warp that walked them together with one elected lane issuing, nothing would tell the compiler that it stays together.)
        uint32_t s = 0, phase = 1, tile_it = 0;
        for (W walk(p, table, ctl, worker, workers); lane == 0 && walk.more(); walk.advance(), ++tile_it) {
            const TurnedPlace at = walk.place(p);
            constexpr int STEP = 16 * CG;
            const int width_cta = (at.rows + STEP - 1) / STEP * 16;
            const int row0 = at.row0 + (CG == 1 ? 0 : static_cast<int>(cta_rank) * width_cta);
            const int n0 = at.col0 + (CG == 1 ? 0 : static_cast<int>(cta_rank) * BM);
            const int boxes = (width_cta + A_CHUNK_ROWS - 1) / A_CHUNK_ROWS;
            // (64-column boxes wholly behind the matrix, as half of the tile is where down has few ranks, are not copied; but one
            // is, so that this lane has a part in every stage)
            const int w_boxes = W_MN ? min(BM / 64, max(1, (p.n - n0 + 63) / 64)) : BM / 64;
            const int w_boxes_other = CG == 1 ? 0 : W_MN ? min(BM / 64, max(1, (p.n - n0 - BM + 63) / 64)) : BM / 64;
            const int bytes = (w_boxes + w_boxes_other) * (S::W_BYTES / (BM / 64)) + CG * S::SUB * boxes * (A_CHUNK_ROWS * BK * 2);
            for (int kb = kb_first; kb < kb_last; ++kb) {
                mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x100 | s);
                uint8_t *w_dst = smem + s * S::STAGE_BYTES;
                uint8_t *x_dst = w_dst + S::W_BYTES;
                if (warp == 0) {
                    if (leader) {
                        // (the issuer of the products learns the tile's rows here: placing a tile takes a few hundred
                        // cycles, which the producer is ahead and the tensor core would idle)
                        if (kb == kb_first) ctl->tile_rows[tile_it % MAX_STAGES] = at.rows;
                        mbar_expect_tx(&ctl->full[s], bytes);
                    }
                    if constexpr (W_MN) {
#pragma unroll
                        for (int j = 0; j < BM / 64; ++j)
                            if (j < w_boxes)
                                load_3d<CG>(w_dst + j * (S::DEPTH * 128), &map_w, &ctl->full[s], n0 + j * 64, kb * S::DEPTH, at.matrix);
                    } else {
#pragma unroll
                        for (int sub = 0; sub < S::SUB; ++sub)
                            load_3d<CG>(w_dst + sub * A_STAGE_BYTES, &map_w, &ctl->full[s], kb * S::DEPTH + sub * BK, n0, at.matrix);
                    }
                } else {
#pragma unroll
                    for (int sub = 0; sub < S::SUB; ++sub) {
                        const int k0 = kb * S::DEPTH + sub * BK;
                        if (boxes == S::ROWS_CTA / A_CHUNK_ROWS) {
                            load_2d<CG>(x_dst + sub * S::X_BYTES, &map_x, &ctl->full[s], k0, row0);
                        } else {
                            for (int c = 0; c < boxes; ++c)
                                load_2d<CG>(x_dst + sub * S::X_BYTES + c * (A_CHUNK_ROWS * BK * 2), &map_x_chunk, &ctl->full[s],
                                            k0, row0 + c * A_CHUNK_ROWS);
                        }
                    }
                }
                if (++s == STAGES) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------- MMA issuer -------------------------------
        // (The warp goes through the loop together: its branches are its votes and values known to be the warp's.  What one lane
        // does alone is a single probe of a barrier, followed by a vote, or a stage's products and their commit, behind an
        // election of their own and before a __syncwarp.  An earlier lora_kernel, whose issuer held one election through loops that
        // the elected lane went through by itself, was seen to issue a commit twice.  Its issuer is a lone lane throughout.)
        if (leader) {
            const uint32_t smem_base = smem_u32(smem);
            uint32_t s = 0, phase = 0, acc_it = 0;
            bool ready = false;
            const int total = __shfl_sync(0xffffffffu, ctl->tiles_m, 0) * p.n_tiles;  // (known to be the warp's)
            for (int tile = worker; tile < total; tile += workers, ++acc_it) {
                constexpr int STEP = 16 * CG;
                uint32_t idesc = 0;
                const uint32_t buf = acc_it & 1;
                mbar_wait_together(&ctl->tmem_empty[buf], ((acc_it >> 1) & 1) ^ 1, wait_ctx, 0x200 | buf);
                tcgen05_fence_after_sync();
                const uint32_t tmem_acc = tmem_base + buf * NT;
                for (int kb = kb_first; kb < kb_last; ++kb) {
                    if (!ready) mbar_wait_together(&ctl->full[s], phase, wait_ctx, 0x300 | s);
                    tcgen05_fence_after_sync();
                    if (kb == kb_first) {
                        const int rows = __shfl_sync(0xffffffffu, ctl->tile_rows[acc_it % MAX_STAGES], 0);
                        idesc = umma_instr_desc(BM * CG, (rows + STEP - 1) / STEP * STEP, p.bf16 != 0, W_MN, false);
                    }
                    const uint32_t w_addr = smem_base + s * S::STAGE_BYTES;
                    const uint32_t x_addr = w_addr + S::W_BYTES;
                    const uint32_t s_next = s + 1 == STAGES ? 0 : s + 1;
                    const uint32_t phase_next = s_next == 0 ? phase ^ 1 : phase;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < S::DEPTH / UMMA_K; ++kk) {
                            const int sub = kk / (BK / UMMA_K), step = kk % (BK / UMMA_K);
                            const uint64_t desc_w =
                                W_MN ? umma_smem_desc(w_addr + kk * (UMMA_K * 128), S::DEPTH * 128, 1024)
                                     : umma_smem_desc(w_addr + sub * A_STAGE_BYTES + step * (UMMA_K * 2), 16, 1024);
                            const uint64_t desc_x = umma_smem_desc(x_addr + sub * S::X_BYTES + step * (UMMA_K * 2), 16, 1024);
                            umma_ss<CG>(tmem_acc, desc_w, desc_x, idesc, (kb != kb_first || kk != 0) ? 1u : 0u);
                        }
                        if constexpr (CG == 1) umma_commit<1>(&ctl->empty[s]);
                        else umma_commit_pair_multicast(&ctl->empty[s], 0x3);
                    }
                    __syncwarp();
                    ready = __all_sync(0xffffffffu, mbar_test_wait(&ctl->full[s_next], phase_next));
                    s = s_next;
                    phase = phase_next;
                }
                if (elect_one()) {
                    if constexpr (CG == 1) umma_commit<1>(&ctl->tmem_full[buf]);
                    else umma_commit_pair_multicast(&ctl->tmem_full[buf], 0x3);
                }
                __syncwarp();
            }
        }
    } else {
        // -------------------------------- epilogue --------------------------------
        const int quadrant = warp & 3;
        const int half = (warp - 2) / 4;
        const int n_lane = quadrant * 32 + lane;
        const bool bf16 = p.bf16 != 0;
        uint32_t acc_it = 0;
        [[maybe_unused]] bool arrived = false;  // at the cluster barrier that ends the kernel
        if constexpr (SPLIT) cluster_wait();
        for (W walk(p, table, ctl, worker, workers); walk.more(); walk.advance(), ++acc_it) {
            const TurnedPlace at = walk.place(p);
            const int n = at.col0 + (CG == 1 ? 0 : static_cast<int>(cta_rank) * BM) + n_lane;
            const uint32_t buf = acc_it & 1;
            if constexpr (FEW)
                adapters_part(p, at, partials, low, static_cast<int>(cta_rank), split);
            mbar_wait(&ctl->tmem_full[buf], (acc_it >> 1) & 1, wait_ctx, 0x400 | buf);
            tcgen05_fence_after_sync();
            const uint32_t taddr = tmem_base + buf * NT + (static_cast<uint32_t>(quadrant * 32) << 16);
            const int64_t column_at = n * p.out_stride1;
            const int n_end = PARTS ? p.rank_blocks * RANK_BLOCK : p.n;
            const float scale = PARTS ? p.scales[at.matrix * p.scales_stride] : 1.f;
            const int share = SPLIT ? split_share(at.rows, split) : 0;
#pragma unroll 1
            for (int t0 = 32 * half; t0 < at.rows; t0 += 64) {
                uint32_t acc[32];
                __syncwarp();
                tmem_ld_32x32(taddr + t0, acc);
                tmem_wait_ld();
                if constexpr (SPLIT) {
                    // four rows at a time to the CTA whose share they are, into this CTA's part there
                    float4 *part = reinterpret_cast<float4 *>(partials) + static_cast<int>(cta_rank) * (share / 4) * BM + n_lane;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (t0 + j >= at.rows) break;
                        const int cta = (t0 + j) / share;
                        float4 *dst = part + (t0 + j - cta * share) / 4 * BM;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (kb_first < kb_last)
                            v = make_float4(__uint_as_float(acc[j]), __uint_as_float(acc[j + 1]), __uint_as_float(acc[j + 2]),
                                            __uint_as_float(acc[j + 3]));
                        if (FEW && cta == static_cast<int>(cta_rank)) {
                            const float4 adapters = *dst;
                            v.x += adapters.x;
                            v.y += adapters.y;
                            v.z += adapters.z;
                            v.w += adapters.w;
                        }
                        store_remote(remote_address(dst, cta), v);
                    }
                } else if constexpr (PARTS) {
                    if (n - lane < n_end && bf16) {
                        uint32_t rest[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float v = n < p.n ? scale * __uint_as_float(acc[j]) : 0.f;
                            const TwoParts parts(v, 8);
                            acc[j] = __float_as_uint(parts.first);
                            rest[j] = __float_as_uint(parts.rest);
                        }
                        uint16_t *block = static_cast<uint16_t *>(p.out) + n / RANK_BLOCK * RANK_BLOCK;
                        const int64_t pitch = 2 * p.out_stride0;
                        store_turned(acc, block, pitch, at.row0 + t0, at.rows - t0, at.row0 + t0 + 16, at.rows - t0 - 16, n, n_end, true);
                        store_turned(rest, block + RANK_BLOCK, pitch, at.row0 + t0, at.rows - t0, at.row0 + t0 + 16, at.rows - t0 - 16, n, n_end, true);
                    } else if (n - lane < n_end) {
                        float *out = static_cast<float *>(p.out) + (at.row0 + t0) * p.out_stride0 + n;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (t0 + j < at.rows) out[j * p.out_stride0] = n < p.n ? scale * __uint_as_float(acc[j]) : 0.f;
                    }
                } else if (p.out_vec) {
                    store_turned(acc, p.out, p.out_stride0, at.row0 + t0, at.rows - t0, at.row0 + t0 + 16, at.rows - t0 - 16, n, p.n, bf16);
                } else if (n < p.n) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (t0 + j < at.rows)
                            store16(p.out, (at.row0 + t0 + j) * p.out_stride0 + column_at, __uint_as_float(acc[j]), bf16);
                }
            }
            if constexpr (SPLIT) {
                __syncwarp();  // (one arrival a warp and CTA, after the stores of all its lanes)
                if (lane < split) mbar_arrive_cluster(&ctl->partials, lane);
                __syncwarp();
                cluster_arrive();
                arrived = true;
                mbar_wait_cluster(&ctl->partials, 0, wait_ctx, 0x500);
                const int first = static_cast<int>(cta_rank) * share, last = min(at.rows, first + share);
                if (n < n_end)
                    for (int t = first + 4 * half; t < last; t += 8) {
                        const float4 *part = reinterpret_cast<const float4 *>(partials) + (t - first) / 4 * BM + n_lane;
                        float sum[4] = {};
#pragma unroll 4
                        for (int cta = 0; cta < split; ++cta) {
                            const float4 v = part[cta * (share / 4) * BM];
                            sum[0] += v.x;
                            sum[1] += v.y;
                            sum[2] += v.z;
                            sum[3] += v.w;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (t + j >= last) break;
                            const int64_t row_at = (at.row0 + t + j) * p.out_stride0;
                            if constexpr (PARTS) {
                                const float v = n < p.n ? scale * sum[j] : 0.f;
                                if (bf16) {
                                    const int64_t to = 2 * row_at + n / RANK_BLOCK * (2 * RANK_BLOCK) + n % RANK_BLOCK;
                                    const TwoParts parts(v, 8);
                                    store16(p.out, to, parts.first, true);
                                    store16(p.out, to + RANK_BLOCK, parts.rest, true);
                                } else {
                                    static_cast<float *>(p.out)[row_at + n] = v;
                                }
                            } else {
                                store16(p.out, row_at + column_at, sum[j], bf16);
                            }
                        }
                    }
            }
            tcgen05_fence_before_sync();
            if (CG == 1 || leader) mbar_arrive(&ctl->tmem_empty[buf]);
            else mbar_arrive_cluster(&ctl->tmem_empty[buf], 0);
        }
        if constexpr (FEW) griddepcontrol_wait();  // (also where there was no tile: what follows this launch may rely on the one before)
        if constexpr (SPLIT) {
            if (!arrived) cluster_arrive();
        }
    }
    if constexpr (SPLIT) {
        if (warp < 2 || warp == ROW_WARP) {
            __syncwarp();
            cluster_wait();
            cluster_arrive();
        }
    }

    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if constexpr (SPLIT) {
        // No CTA leaves while another may still write into its memory.  (The epilogue has arrived early: what is left
        // of its work is its own CTA's.)
        cluster_wait();
    }
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc<CG>(tmem_base, TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------
// The shared projection with adapters beside it, for many rows, with the operands exchanged as in turned_kernel.  The rows
// stand in a padded space of accumulator columns in which every request starts at a multiple of 16 (32); a tile is NT columns of
// it, whatever requests they belong to, against 128 (256) columns of rhs.  Then, for every request with an adapter that has
// columns in the tile, its second product is an ordinary product into just these columns, 32 ranks a stage: nothing of one
// request's adapter, infinities and NaN included, meets another's columns.  (scales lhs . down) comes from the launch before, under
// which this one starts.
//
// WIDE (fp16): two fp16 parts would hold neither values above 65504 nor the low parts of small ones, so the value comes in 32
// bits, and four warps split it into two operands of eleven bits and eight of exponent (kind::tf32), and widen up to a third, once
// the copies have landed.  Products of such operands take twice as long, and the tile's end waits for the warps: bf16, whose two
// parts have the range of fp32, would lose 6 % by it at 8192 rows of 6 requests (4096 x 4096, rank 32: 239 and 254 us) and 15 % at
// 4096 rows towards the input (4096 x 2048, rank 64: 81.5 and 93.8).
//
// What bounds it: for long requests the products of the projection and the board's power, as in turned_kernel: 8192 rows of 6
// requests, 4096 x 4096, rank 32, take 242 us back to back (1.16 PFLOP/s; fp16 267), some 15 of them the launch before, which
// reads lhs once more.  For short ones the padding (rank 16): 2048 rows of 256 requests take 209 us, of 64 75.  Small calls are
// latency: of the 37 us of 1533 rows of 40 requests (1000 x 2056, rank 24, fp16) 10 are the launch before, 5 this one's table and
// first copies.
// ---------------------------------------------------------------------------
// The columns [from, to) of the padded space that a run of the table (tiles_before: its first column) has in [low, high).
template <int STEP>
struct Piece {
    int from, to;
    __device__ Piece(const Run &run, int low, int high)
        : from(max(run.tiles_before, low)), to(min(run.tiles_before + (run.end - run.begin + STEP - 1) / STEP * STEP, high)) {}
    __device__ int row(const Run &run) const { return run.begin + from - run.tiles_before; }
};

// One operand of a second product, 128 columns of up and 32 ranks, in 32 bits as a K-major tile of 128-byte swizzle rows: exact for
// either type.  `raw` holds the ranks as rows (MN: two boxes of 64 columns) or the columns (64 ranks each, the first 32 count).
// Threads go through it in an order in which eight neighbours read and write different banks.
template <bool MN>
__device__ __forceinline__ void widen_up(const uint8_t *raw, uint8_t *wide, int thread, bool bf16) {
    const auto put = [&](int column, int chunk, float a, float b, float c, float d) {  // four ranks of a column
        *reinterpret_cast<float4 *>(wide + column * 128 + ((chunk ^ (column & 7)) << 4)) = make_float4(a, b, c, d);
    };
    if constexpr (MN) {  // four ranks of eight columns
        static_assert(SPLITTERS * 32 == BM / 8 * RANK_BLOCK / 4, "one task a thread");
        const int q = thread & 7, c = (thread >> 3) ^ (q >> 1);
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rank = 4 * q + i;
            v[i] = *reinterpret_cast<const uint4 *>(raw + (c >> 3) * (RANK_BLOCK * 128) + rank * 128 + (((c & 7) ^ (rank & 7)) << 4));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const auto at = [&](const uint4 &w) { return half_of(j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w, j & 1, bf16); };
            put(c * 8 + j, q, at(v[0]), at(v[1]), at(v[2]), at(v[3]));
        }
    } else {  // eight ranks of a column
#pragma unroll
        for (int task = thread; task < BM * (RANK_BLOCK / 8); task += SPLITTERS * 32) {
            const int column = task / 32 * 8 + (task & 7), c = (task >> 3) & 3;
            const uint4 v = *reinterpret_cast<const uint4 *>(raw + column * 128 + ((c ^ (column & 7)) << 4));
            put(column, 2 * c, half_of(v.x, 0, bf16), half_of(v.x, 1, bf16), half_of(v.y, 0, bf16), half_of(v.y, 1, bf16));
            put(column, 2 * c + 1, half_of(v.z, 0, bf16), half_of(v.z, 1, bf16), half_of(v.w, 0, bf16), half_of(v.w, 1, bf16));
        }
    }
}

// The other operand, (scales lhs . down) of `rows` rows and 32 ranks, as two numbers of eleven bits each, which is what the
// products keep of a 32-bit operand: the value's first eleven and the rest, rounded, 2^-22 of the value off at most.  The first
// take the value's place, the second lie `second` bytes behind.
__device__ __forceinline__ void split_low(uint8_t *values, int second, int rows, int thread) {
    for (int i = thread; i < rows * (RANK_BLOCK / 4); i += SPLITTERS * 32) {
        float4 *at = reinterpret_cast<float4 *>(values) + i;
        const auto rounded = [](float v) {
            uint32_t bits;
            asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(bits) : "f"(v));
            return __uint_as_float(bits);
        };
        const float4 v = *at;
        const TwoParts x(v.x, 11), y(v.y, 11), z(v.z, 11), w(v.w, 11);
        *at = make_float4(x.first, y.first, z.first, w.first);
        *reinterpret_cast<float4 *>(values + second + i * 16) =
            make_float4(rounded(x.rest), rounded(y.rest), rounded(z.rest), rounded(w.rest));
    }
}

// The run that holds a column.
__device__ __forceinline__ int run_at(const Run *table, int runs, int column) {
    int low = 0, high = runs - 1;
    while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (table[mid].tiles_before <= column) low = mid;
        else high = mid - 1;
    }
    return low;
}

template <int CG, int NT, bool W_MN, bool WIDE>
__global__ void __launch_bounds__(lora_threads(WIDE), 1)
    lora_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                const __grid_constant__ CUtensorMap map_x32, const __grid_constant__ CUtensorMap map_x16,
                const __grid_constant__ CUtensorMap map_low, const __grid_constant__ CUtensorMap map_up,
                const __grid_constant__ Params p) {
    using S = Turned<CG, NT>;
    constexpr int STAGES = S::STAGES;
    constexpr int ROW_BYTES = BK * 2;  // of one row in a 64-deep block
    constexpr int UP_CG = WIDE ? 1 : CG;  // (what warps of the CTA work on arrives at a barrier of the CTA)
    constexpr int UP_AT = S::W_BYTES - BM * RANK_BLOCK * 4;  // where a stage holds up in 32 bits, behind what the copies bring
    static_assert(UP_AT >= A_STAGE_BYTES && UP_AT % 1024 == 0, "a stage of ranks");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Control *ctl = reinterpret_cast<Control *>(smem + STAGES * S::STAGE_BYTES);
    Run *table = reinterpret_cast<Run *>(reinterpret_cast<uint8_t *>(ctl) + CONTROL_BYTES);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const WaitCtx wait_ctx{&ctl->abort_flag, p.status, KID_GROUPED};
    const uint32_t cta_rank = CG == 1 ? 0u : cluster_cta_rank();
    const bool leader = cta_rank == 0;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&ctl->full[s], 1 + ROW_PRODUCERS * CG);
            mbar_init(&ctl->empty[s], 1);
            mbar_init(&ctl->raw[s], 1);
            mbar_init(&ctl->clean[s], SPLITTERS * CG);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], EPILOGUE_WARPS * 32 * CG);
        }
        ctl->abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_low);
        tma_prefetch_desc(&map_up);
    }
    if (warp == 1) {
        tmem_alloc<CG>(&ctl->tmem_base, TMEM_COLS);
        tmem_relinquish<CG>();
    }
    constexpr int STEP = 16 * CG;  // columns of a request start at multiples of it (a product of a pair takes steps of 32)
    build_table<true>(p, table, ctl, STEP);
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    const int runs = __shfl_sync(0xffffffffu, ctl->runs, 0);
    const int columns = __shfl_sync(0xffffffffu, ctl->tiles_m, 0) * STEP;  // of the padded space
    const int m_tiles = (columns + NT - 1) / NT, total = m_tiles * p.n_tiles;

    // (lone lanes, as in turned_kernel)
    if (warp == 0 && lane == 0) {
        // ------------------- TMA producer of the matrices, rhs and up -------------------
        uint32_t s = 0, phase = 1;
        const auto next = [&] {
            if (++s == STAGES) {
                s = 0;
                phase ^= 1;
            }
        };
        const int up_bytes = p.up_mn ? BM * RANK_BLOCK * 2 : A_STAGE_BYTES;
        for (int tile = worker; tile < total; tile += workers) {
            int m, n;
            raster(tile, m_tiles, p.n_tiles, p.group_m, m, n);
            const int first = m * NT, last = min(first + NT, columns);
            const int n0 = n * S::TILE_N + static_cast<int>(cta_rank) * BM;
            // (the even CTA's barriers count the bytes of both)
            const int bytes = CG * S::W_BYTES + S::SUB * (last - first) * ROW_BYTES;
            for (int kb = 0; kb < p.k_blocks; ++kb) {
                mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x100 | s);
                uint8_t *dst = smem + s * S::STAGE_BYTES;
                if (leader) mbar_expect_tx(&ctl->full[s], bytes);
                if constexpr (W_MN) {
#pragma unroll
                    for (int j = 0; j < BM / 64; ++j)
                        load_3d<CG>(dst + j * (S::DEPTH * 128), &map_w, &ctl->full[s], n0 + j * 64, kb * S::DEPTH, 0);
                } else {
#pragma unroll
                    for (int sub = 0; sub < S::SUB; ++sub)
                        load_3d<CG>(dst + sub * A_STAGE_BYTES, &map_w, &ctl->full[s], kb * S::DEPTH + sub * BK, n0, 0);
                }
                next();
            }
            for (int r = run_at(table, runs, first); r < runs && table[r].tiles_before < last; ++r) {
                const int matrix = table[r].matrix;
                if (matrix < 0) continue;
                for (int rb = 0; rb < p.rank_blocks; ++rb) {
                    mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x110 | s);
                    uint8_t *dst = smem + s * S::STAGE_BYTES;
                    if constexpr (WIDE) {
                        mbar_expect_tx(&ctl->raw[s], up_bytes + S::X_BYTES);
                        if (leader) mbar_arrive(&ctl->full[s]);  // (keeps its phases in step; the issuer waits for `clean` too)
                    } else if (leader) {
                        mbar_expect_tx(&ctl->full[s], CG * (up_bytes + S::X_BYTES));
                    }
                    uint64_t *bar = WIDE ? &ctl->raw[s] : &ctl->full[s];
                    if (p.up_mn) {
#pragma unroll
                        for (int j = 0; j < BM / 64; ++j)
                            load_3d<UP_CG>(dst + j * (RANK_BLOCK * 128), &map_up, bar, n0 + j * 64, rb * RANK_BLOCK, matrix);
                    } else {
                        load_3d<UP_CG>(dst, &map_up, bar, rb * RANK_BLOCK, n0, matrix);
                    }
                    next();
                }
            }
        }
    } else if (warp >= ROW_WARP && warp < SPLIT_WARP && lane == 0) {
        // -------------- TMA producers of the rows, of lhs and of (scales lhs . down) --------------
        // Where requests meet in a tile its rows are many small boxes: one lane's copies of them took 2300 cycles a stage, over
        // twice the products' time.  Four lanes share them: the halves of a stage, and every other box.
        const int sub = (warp - ROW_WARP) & 1, turn = (warp - ROW_WARP) >> 1;
        constexpr int BOXES = S::ROWS_CTA / 16 / 2;  // most of one lane
        bool waited = false;
        const auto wait_parts = [&] {  // for the kernel before this one, under which this one starts
            griddepcontrol_wait();
            fence_proxy_async();  // (it wrote, copies read)
            waited = true;
        };
        uint32_t s = 0, phase = 1;
        const auto next = [&] {  // (a stage that a lane copies nothing of may not be filled and emptied without it: see Control)
            if (leader) mbar_arrive(&ctl->full[s]);
            else arrive_leader(&ctl->full[s]);
            if (++s == STAGES) {
                s = 0;
                phase ^= 1;
            }
        };
        for (int tile = worker; tile < total; tile += workers) {
            int m, n;
            raster(tile, m_tiles, p.n_tiles, p.group_m, m, n);
            const int first = m * NT, last = min(first + NT, columns);
            // this CTA's columns: half of the tile's for one of a pair
            const int width_cta = (last - first + STEP - 1) / STEP * 16;
            const int mine = first + static_cast<int>(cta_rank) * width_cta, mine_end = min(mine + width_cta, last);
            const int run_first = run_at(table, runs, first), run_mine = run_at(table, runs, mine);
            // this lane's boxes, found once a tile (the walk of the requests costs as much as the copies): where each begins in
            // lhs and in a stage, and, in the offset's last bits, how many rows it has
            int box_row[BOXES], box_at[BOXES], boxes = 0, box = 0;
            for (int r = run_mine; r < runs && table[r].tiles_before < mine_end; ++r) {
                const Piece<STEP> piece(table[r], mine, mine_end);
                const int row = piece.row(table[r]), count = piece.to - piece.from;
                for (int c = 0; c < count; ++box) {
                    const int size = count == S::ROWS_CTA ? S::ROWS_CTA : count - c >= 32 ? 32 : 16;
                    if ((box & 1) == turn) {
#pragma unroll
                        for (int i = 0; i < BOXES; ++i)
                            if (i == boxes) {
                                box_row[i] = row + c;
                                box_at[i] = (piece.from - mine + c) * ROW_BYTES + size;
                            }
                        ++boxes;
                    }
                    c += size;
                }
            }
            for (int kb = 0; kb < p.k_blocks; ++kb) {
                mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x120 | s);
                uint8_t *dst = smem + s * S::STAGE_BYTES + S::W_BYTES + sub * S::X_BYTES;
                const int k0 = kb * S::DEPTH + sub * BK;
#pragma unroll
                for (int i = 0; i < BOXES; ++i)
                    if (i < boxes) {
                        const int size = box_at[i] & (ROW_BYTES * 2 - 1);
                        uint8_t *at = dst + (box_at[i] - size);
                        if (size == 16) load_2d<CG>(at, &map_x16, &ctl->full[s], k0, box_row[i]);
                        else if (size == 32) load_2d<CG>(at, &map_x32, &ctl->full[s], k0, box_row[i]);
                        else load_2d<CG>(at, &map_x, &ctl->full[s], k0, box_row[i]);
                    }
                next();
            }
            for (int r = run_first; r < runs && table[r].tiles_before < last; ++r) {
                if (table[r].matrix < 0) continue;
                const Piece<STEP> piece(table[r], first, last);
                // a pair's CTAs bring half of the piece each (and what follows it, unused)
                const int row = piece.row(table[r]) + static_cast<int>(cta_rank) * ((piece.to - piece.from) / CG);
                for (int rb = 0; rb < p.rank_blocks; ++rb) {
                    mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x130 | s);
                    uint8_t *dst = smem + s * S::STAGE_BYTES + S::W_BYTES;
                    if (warp == ROW_WARP) {
                        if (!waited) wait_parts();
                        load_2d<UP_CG>(dst, &map_low, WIDE ? &ctl->raw[s] : &ctl->full[s], rb * (WIDE ? RANK_BLOCK : BK), row);
                    }
                    next();
                }
            }
        }
        if (warp == ROW_WARP && !waited) wait_parts();  // (what follows this launch may rely on the one before)
    } else if (warp == 1) {
        // ------------------------------- MMA issuer -------------------------------
        if (leader && lane == 0) {
            const uint32_t smem_base = smem_u32(smem);
            const uint32_t up_step = p.up_mn ? UMMA_K * 128 : UMMA_K * 2, up_lbo = p.up_mn ? RANK_BLOCK * 128 : 16;
            uint32_t s = 0, phase = 0, acc_it = 0;
            [[maybe_unused]] uint32_t clean_phases = 0;  // (a bit a stage, as in grad_kernel)
            bool ready = false;
            for (int tile = worker; tile < total; tile += workers, ++acc_it) {
                int m, n;
                raster(tile, m_tiles, p.n_tiles, p.group_m, m, n);
                const int first = m * NT, last = min(first + NT, columns);
                const uint32_t idesc = umma_instr_desc(BM * CG, (last - first + STEP - 1) / STEP * STEP, p.bf16 != 0, W_MN, false);
                const uint32_t buf = acc_it & 1;
                mbar_wait(&ctl->tmem_empty[buf], ((acc_it >> 1) & 1) ^ 1, wait_ctx, 0x200 | buf);
                tcgen05_fence_after_sync();
                const uint32_t tmem_acc = tmem_base + buf * NT;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!ready) mbar_wait(&ctl->full[s], phase, wait_ctx, 0x300 | s);
                    tcgen05_fence_after_sync();
                    const uint32_t w_addr = smem_base + s * S::STAGE_BYTES;
                    const uint32_t x_addr = w_addr + S::W_BYTES;
                    const uint32_t s_next = s + 1 == STAGES ? 0 : s + 1;
                    const uint32_t phase_next = s_next == 0 ? phase ^ 1 : phase;
#pragma unroll
                    for (int kk = 0; kk < S::DEPTH / UMMA_K; ++kk) {
                        const int sub = kk / (BK / UMMA_K), step = kk % (BK / UMMA_K);
                        const uint64_t desc_w =
                            W_MN ? umma_smem_desc(w_addr + kk * (UMMA_K * 128), S::DEPTH * 128, 1024)
                                 : umma_smem_desc(w_addr + sub * A_STAGE_BYTES + step * (UMMA_K * 2), 16, 1024);
                        const uint64_t desc_x = umma_smem_desc(x_addr + sub * S::X_BYTES + step * (UMMA_K * 2), 16, 1024);
                        umma_ss<CG>(tmem_acc, desc_w, desc_x, idesc, (kb != 0 || kk != 0) ? 1u : 0u);
                        if (kk == S::DEPTH / UMMA_K / 2 - 1)
                            ready = mbar_test_wait(&ctl->full[s_next], phase_next);
                    }
                    if constexpr (CG == 1) umma_commit<1>(&ctl->empty[s]);
                    else umma_commit_pair_multicast(&ctl->empty[s], 0x3);
                    s = s_next;
                    phase = phase_next;
                }
                // (Products of one shape into the same accumulator follow one another in the order of their issue, products of
                // different shapes need not: the second products wait until the projection's have ended, which is when its
                // last stage is empty.)
                bool ended = false;
                const uint32_t s_last = s == 0 ? STAGES - 1 : s - 1, phase_last = s == 0 ? phase ^ 1 : phase;
                for (int r = run_at(table, runs, first); r < runs && table[r].tiles_before < last; ++r) {
                    if (table[r].matrix < 0) continue;
                    if (!ended) {
                        mbar_wait(&ctl->empty[s_last], phase_last, wait_ctx, 0x800 | s_last);
                        tcgen05_fence_after_sync();
                        ended = true;
                    }
                    const Piece<STEP> piece(table[r], first, last);
                    const uint32_t idesc_up = WIDE ? umma_instr_desc_tf32(BM * CG, piece.to - piece.from)
                                                   : umma_instr_desc(BM * CG, piece.to - piece.from, p.bf16 != 0, p.up_mn != 0, false);
                    const uint32_t tmem_piece = tmem_acc + (piece.from - first);
                    for (int rb = 0; rb < p.rank_blocks; ++rb) {
                        mbar_wait(&ctl->full[s], phase, wait_ctx, 0x310 | s);
                        if constexpr (WIDE) {
                            mbar_wait_cluster(&ctl->clean[s], (clean_phases >> s) & 1, wait_ctx, 0x700 | s);
                            clean_phases ^= 1u << s;
                        }
                        tcgen05_fence_after_sync();
                        const uint32_t stage = smem_base + s * S::STAGE_BYTES, low_addr = stage + S::W_BYTES;
                        constexpr int STEP_K = WIDE ? 8 : UMMA_K;
                        const int steps = (min(RANK_BLOCK, p.rank - rb * RANK_BLOCK) + STEP_K - 1) / STEP_K;
                        for (int kk = 0; kk < steps; ++kk) {
                            const uint64_t desc_up = WIDE ? umma_smem_desc(stage + UP_AT + kk * 32, 16, 1024) : umma_smem_desc(stage + kk * up_step, up_lbo, 1024);
#pragma unroll
                            for (int part = 0; part < 2; ++part) {
                                if constexpr (WIDE)
                                    umma_ss_tf32<CG>(tmem_piece, desc_up, umma_smem_desc(low_addr + part * S::X_BYTES + kk * 32, 16, 1024), idesc_up, 1u);
                                else
                                    umma_ss<CG>(tmem_piece, desc_up, umma_smem_desc(low_addr + part * (RANK_BLOCK * 2) + kk * (UMMA_K * 2), 16, 1024), idesc_up, 1u);
                            }
                        }
                        if constexpr (CG == 1) umma_commit<1>(&ctl->empty[s]);
                        else umma_commit_pair_multicast(&ctl->empty[s], 0x3);
                        if (++s == STAGES) {
                            s = 0;
                            phase ^= 1;
                        }
                    }
                }
                ready = false;
                if constexpr (CG == 1) umma_commit<1>(&ctl->tmem_full[buf]);
                else umma_commit_pair_multicast(&ctl->tmem_full[buf], 0x3);
            }
        }
    } else if (WIDE && warp >= SPLIT_WARP) {
        // ------------- the adapters' operands: up in 32 bits, (scales lhs . down) in two parts -------------
        const int thread = static_cast<int>(threadIdx.x) - SPLIT_WARP * 32;
        const bool bf16 = p.bf16 != 0;
        uint32_t it = 0, phases = 0;  // stages so far; a phase bit a stage
        for (int tile = worker; tile < total; tile += workers) {
            int m, n;
            raster(tile, m_tiles, p.n_tiles, p.group_m, m, n);
            const int first = m * NT, last = min(first + NT, columns);
            it += p.k_blocks;
            for (int r = run_at(table, runs, first); r < runs && table[r].tiles_before < last; ++r) {
                if (table[r].matrix < 0) continue;
                const Piece<STEP> piece(table[r], first, last);
                for (int rb = 0; rb < p.rank_blocks; ++rb, ++it) {
                    const uint32_t s = it % STAGES;
                    mbar_wait_warp(&ctl->raw[s], (phases >> s) & 1, wait_ctx, 0x600 | s);
                    phases ^= 1u << s;
                    uint8_t *stage = smem + s * S::STAGE_BYTES;
                    if (p.up_mn) widen_up<true>(stage, stage + UP_AT, thread, bf16);
                    else widen_up<false>(stage, stage + UP_AT, thread, bf16);
                    split_low(stage + S::W_BYTES, S::X_BYTES, (piece.to - piece.from) / CG, thread);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (leader) mbar_arrive(&ctl->clean[s]);
                        else mbar_arrive_cluster(&ctl->clean[s], 0);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= 2 && warp < ROW_WARP) {
        // -------------------------------- epilogue --------------------------------
        const int quadrant = warp & 3, half = (warp - 2) / 4;
        const bool bf16 = p.bf16 != 0;
        uint32_t acc_it = 0;
        for (int tile = worker; tile < total; tile += workers, ++acc_it) {
            int m, n_tile;
            raster(tile, m_tiles, p.n_tiles, p.group_m, m, n_tile);
            const int first = m * NT, last = min(first + NT, columns);
            const int n = n_tile * S::TILE_N + static_cast<int>(cta_rank) * BM + quadrant * 32 + lane;
            const uint32_t buf = acc_it & 1;
            int r = run_at(table, runs, first + 32 * half);
            mbar_wait(&ctl->tmem_full[buf], (acc_it >> 1) & 1, wait_ctx, 0x400 | buf);
            tcgen05_fence_after_sync();
            const uint32_t taddr = tmem_base + buf * NT + (static_cast<uint32_t>(quadrant * 32) << 16);
#pragma unroll 1
            for (int c0 = first + 32 * half; c0 < last; c0 += 64) {
                uint32_t acc[32];
                __syncwarp();
                tmem_ld_32x32(taddr + (c0 - first), acc);
                tmem_wait_ld();
                // two times sixteen columns, each of one request: their first rows, and how many are rows
                int row[2], rows[2];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int c = c0 + 16 * g;
                    while (r + 1 < runs && table[r + 1].tiles_before <= c) ++r;
                    row[g] = table[r].begin + c - table[r].tiles_before;
                    rows[g] = c < last ? min(16, table[r].end - row[g]) : 0;
                }
                if (p.out_vec) {
                    store_turned(acc, p.out, p.out_stride0, row[0], rows[0], row[1], rows[1], n, p.n, bf16);
                } else if (n < p.n) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (j % 16 < rows[j / 16])
                            store16(p.out, (row[j / 16] + j % 16) * p.out_stride0 + n * p.out_stride1, __uint_as_float(acc[j]), bf16);
                }
            }
            tcgen05_fence_before_sync();
            if (CG == 1 || leader) mbar_arrive(&ctl->tmem_empty[buf]);
            else mbar_arrive_cluster(&ctl->tmem_empty[buf], 0);
        }
    }

    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc<CG>(tmem_base, TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------
// Gradient of the matrices: rhs_grad[e] = lhs_e^T . output_grad_e, the reduction runs over the rows of run e.
// Both operands are read where they lie, rows of the reduction first ("MN-major" tiles of 64 rows).  A run's last
// 64-row block also brings rows of the next run: whole 16-row steps behind the run are not issued, and the rest of the
// last step is overwritten with zeros in BOTH operands (a zero in one alone would let a NaN or an infinity of the
// neighbouring run through).
//
// What bounds it: for long runs the products, but not they alone: 16384 rows in 16 runs, 2048 x 4096, take 220 us in a short
// burst, 14 more than as many products forward, with the tensor pipe at work 67 % of the time against 79 %, and 264 (1.0 PFLOP/s)
// back to back, under the board's power limit; 16 equal dense products as a library's batch 235.  For short ones: 61 runs of 33
// rows, 1024 x 776, take 46 us, of which a fill of the gradient takes 26; every tile is one ragged block that goes through copy,
// clearing, products and stores in turn.
// ---------------------------------------------------------------------------
struct GradParams {
    Offsets offsets;
    int rows, m, n;  // rows of the reduction (all runs), lhs columns, output_grad columns
    int m_tiles, n_tiles;
    int bf16;
    void *out;
    int64_t out_stride0, out_stride1, out_batch_stride;
    int out_vec;
    unsigned int *status;
};

// Run e's rows, by the same rule as build_table: bounds clamped by a running maximum.  starts has runs + 1 entries.
__device__ __forceinline__ void build_starts(const Offsets &offsets, int rows, int *starts) {
    for (int i = threadIdx.x; i <= offsets.runs; i += blockDim.x)
        starts[i] = load_index(offsets.data, offsets.stride, offsets.wide, i, 0, rows);
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int bound = 0;
    for (int base = 0; base <= offsets.runs; base += 32) {
        int v = base + lane <= offsets.runs ? starts[base + lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v = max(v, other);
        }
        v = max(v, bound);
        if (base + lane <= offsets.runs) starts[base + lane] = v;
        bound = __shfl_sync(0xffffffffu, v, 31);
    }
}

// Two shapes: 256 x 256 tiles on CTA pairs, whose CTAs each bring 128 columns of either operand, and 128 x 128 tiles on
// single CTAs for gradients with few tiles.  Warp 0 copies lhs, warp 1 issues the products, warps 2 to 9 are the epilogue,
// warp 10 copies output_grad.
//
// In a pair the even CTA's barriers count both CTAs' copies, but each CTA has to overwrite its own rows: a ragged block is
// therefore copied against a barrier of its own in each CTA (`raw`), whose warp 11 overwrites the rows, ahead of the
// issuer like the copies, and arrives at the barrier that the issuer waits for (`clean`, in the even CTA).
constexpr int OUT_BOX_BYTES = 32 * 64;  // 32 rows of 32 columns; two an epilogue warp, so that filling one hides the other's store

template <int CG, int BN>
struct Grad {
    static constexpr int BN_CTA = BN / CG;
    static constexpr int STAGE_BYTES = A_STAGE_BYTES + BN_CTA * BK * 2;
    static constexpr int STAGES = 5;
    static constexpr int TILE_M = BM * CG;
    static constexpr int BOX_BYTES = BK * 128;  // 64 rows of 64 columns
    static constexpr int OUT_BYTES = EPILOGUE_WARPS * 2 * OUT_BOX_BYTES;
};

template <int CG, int BN>
constexpr size_t grad_smem(int runs) {
    return 1024 + Grad<CG, BN>::STAGES * Grad<CG, BN>::STAGE_BYTES + Grad<CG, BN>::OUT_BYTES + CONTROL_BYTES +
           static_cast<size_t>(runs + 1) * 4;
}

struct GradTile {
    int run, m0, n0, length, begin;
};

// Tiles of a run follow one another with the rows of the gradient fastest, so that CTAs at work share panels.
__device__ __forceinline__ GradTile grad_tile(const GradParams &p, const int *starts, int tile, int tile_m, int tile_n) {
    const int per_run = p.m_tiles * p.n_tiles;
    const int run = tile / per_run, inside = tile - run * per_run;
    const int n = inside / p.m_tiles;
    return {run, (inside - n * p.m_tiles) * tile_m, n * tile_n, starts[run + 1] - starts[run], starts[run]};
}

template <int CG, int BN>
__global__ void __launch_bounds__(GRAD_THREADS, 1)
    grad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ GradParams p) {
    using S = Grad<CG, BN>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *boxes = smem + STAGES * S::STAGE_BYTES;
    Control *ctl = reinterpret_cast<Control *>(boxes + S::OUT_BYTES);
    int *starts = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(ctl) + CONTROL_BYTES);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const WaitCtx wait_ctx{&ctl->abort_flag, p.status, KID_GROUPED_GRAD};
    const uint32_t cta_rank = CG == 1 ? 0u : cluster_cta_rank();
    const bool leader = cta_rank == 0;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
            mbar_init(&ctl->raw[s], 1);
            mbar_init(&ctl->clean[s], CG);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->tmem_full[b], 1);
            mbar_init(&ctl->tmem_empty[b], EPILOGUE_WARPS * 32 * CG);
        }
        ctl->abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
        tma_prefetch_desc(&map_out);
    }
    if (warp == 1) {
        tmem_alloc<CG>(&ctl->tmem_base, TMEM_COLS);
        tmem_relinquish<CG>();
    }
    build_starts(p.offsets, p.rows, starts);
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    const int total = p.offsets.runs * p.m_tiles * p.n_tiles;

    // The copies of one operand, COLS columns of it a CTA.  (The tensor map has to be known here: chosen at run time, its
    // address is no constant, and a copy costs several times as much to issue.)
    const auto produce = [&](const CUtensorMap &map, auto cols, auto of_lhs) {
        constexpr int COLS = decltype(cols)::value;
        constexpr bool LHS = decltype(of_lhs)::value;
        uint32_t s = 0, phase = 1;
        if (lane != 0) return;  // (a lone lane, as in turned_kernel)
        for (int tile = worker; tile < total; tile += workers) {
            const GradTile at = grad_tile(p, starts, tile, S::TILE_M, BN);
            const int col0 = (LHS ? at.m0 : at.n0) + static_cast<int>(cta_rank) * COLS;
            for (int k0 = 0; k0 < at.length; k0 += BK) {
                mbar_wait(&ctl->empty[s], phase, wait_ctx, 0x100 | s);
                uint8_t *dst = smem + s * S::STAGE_BYTES + (LHS ? 0 : A_STAGE_BYTES);
                const bool ragged = at.length - k0 < BK && (at.length & (UMMA_K - 1)) != 0;
                if (ragged) {
                    if (LHS) {
                        mbar_expect_tx(&ctl->raw[s], S::STAGE_BYTES);
                        if (leader) mbar_arrive(&ctl->full[s]);  // (keeps its phases in step; the issuer waits for `clean` too)
                    }
#pragma unroll
                    for (int j = 0; j < COLS / 64; ++j)
                        tma_load_2d(dst + j * S::BOX_BYTES, &map, &ctl->raw[s], col0 + j * 64, at.begin + k0);
                } else {
                    if (LHS && leader) mbar_expect_tx(&ctl->full[s], S::STAGE_BYTES * CG);
#pragma unroll
                    for (int j = 0; j < COLS / 64; ++j)
                        load_2d<CG>(dst + j * S::BOX_BYTES, &map, &ctl->full[s], col0 + j * 64, at.begin + k0);
                }
                if (++s == STAGES) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    };

    if (warp == 0) {
        produce(map_a, std::integral_constant<int, BM>(), std::true_type());
    } else if (warp == ROW_WARP) {
        produce(map_b, std::integral_constant<int, S::BN_CTA>(), std::false_type());
    } else if (warp == 1) {
        // ------------------------------- MMA issuer -------------------------------
        const uint32_t idesc = umma_instr_desc(BM * CG, BN, p.bf16 != 0, true, true);
        const uint32_t smem_base = smem_u32(smem);
        uint32_t s = 0, phase = 0, acc_it = 0, clean_phases = 0;  // (a bit a stage: not every use of a stage is ragged)
        bool ready = false;
        for (int tile = leader ? worker : total; tile < total; tile += workers) {
            const int length = __shfl_sync(0xffffffffu, grad_tile(p, starts, tile, S::TILE_M, BN).length, 0);
            if (length == 0) continue;  // (the epilogue stores zeros by itself)
            const int blocks = (length + BK - 1) / BK;
            const uint32_t buf = acc_it & 1;
            mbar_wait_together(&ctl->tmem_empty[buf], ((acc_it >> 1) & 1) ^ 1, wait_ctx, 0x200 | buf);
            ++acc_it;
            tcgen05_fence_after_sync();
            const uint32_t tmem_acc = tmem_base + buf * BN;
            for (int kb = 0; kb < blocks; ++kb) {
                if (!ready) mbar_wait_together(&ctl->full[s], phase, wait_ctx, 0x300 | s);
                const int left = length - kb * BK;
                if (left < BK && (left & (UMMA_K - 1)) != 0) {
                    mbar_wait_together<true>(&ctl->clean[s], (clean_phases >> s) & 1, wait_ctx, 0x700 | s);
                    clean_phases ^= 1u << s;
                }
                tcgen05_fence_after_sync();
                const int steps = left >= BK ? BK / UMMA_K : (left + UMMA_K - 1) / UMMA_K;
                const uint32_t a_addr = smem_base + s * S::STAGE_BYTES;
                const uint32_t b_addr = a_addr + A_STAGE_BYTES;
                const uint32_t s_next = s + 1 == STAGES ? 0 : s + 1;
                const uint32_t phase_next = s_next == 0 ? phase ^ 1 : phase;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                        const uint64_t desc_a = umma_smem_desc(a_addr + kk * (UMMA_K * 128), S::BOX_BYTES, 1024);
                        const uint64_t desc_b = umma_smem_desc(b_addr + kk * (UMMA_K * 128), S::BOX_BYTES, 1024);
                        if (kk < steps) umma_ss<CG>(tmem_acc, desc_a, desc_b, idesc, (kb != 0 || kk != 0) ? 1u : 0u);
                    }
                    if constexpr (CG == 1) umma_commit<1>(&ctl->empty[s]);
                    else umma_commit_pair_multicast(&ctl->empty[s], 0x3);
                }
                __syncwarp();
                ready = __all_sync(0xffffffffu, mbar_test_wait(&ctl->full[s_next], phase_next));
                s = s_next;
                phase = phase_next;
            }
            if (elect_one()) {
                if constexpr (CG == 1) umma_commit<1>(&ctl->tmem_full[buf]);
                else umma_commit_pair_multicast(&ctl->tmem_full[buf], 0x3);
            }
            __syncwarp();
        }
    } else if (warp == ROW_WARP + 1) {
        // --------------- the rows behind a run in its last block ---------------
        uint32_t it = 0, phases = 0;  // blocks so far; a phase bit a stage (not every use of a stage is ragged)
        for (int tile = worker; tile < total; tile += workers) {
            const int length = grad_tile(p, starts, tile, S::TILE_M, BN).length;
            it += (length + BK - 1) / BK;
            if ((length & (UMMA_K - 1)) == 0) continue;
            const uint32_t s = (it - 1) % STAGES, phase = (phases >> s) & 1;
            phases ^= 1u << s;
            mbar_wait_warp(&ctl->raw[s], phase, wait_ctx, 0x600 | s);
            const int first = length & (BK - 1), chunks = (UMMA_K - (length & (UMMA_K - 1))) * 8;  // 16-byte chunks of a box
            uint8_t *rows = smem + s * S::STAGE_BYTES + first * 128;
            for (int i = lane; i < chunks; i += 32)
#pragma unroll
                for (int b = 0; b < (BM + S::BN_CTA) / 64; ++b)
                    *reinterpret_cast<uint4 *>(rows + b * S::BOX_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(&ctl->clean[s]);
                else mbar_arrive_cluster(&ctl->clean[s], 0);
            }
            __syncwarp();
        }
    } else {
        // -------------------------------- epilogue --------------------------------
        const int quadrant = warp & 3, half = (warp - 2) / 4;
        const bool bf16 = p.bf16 != 0;
        uint32_t box_it = 0;
        uint32_t acc_it = 0;
        for (int tile = worker; tile < total; tile += workers) {
            const GradTile at = grad_tile(p, starts, tile, S::TILE_M, BN);
            const int row0 = at.m0 + static_cast<int>(cta_rank) * BM + quadrant * 32, row = row0 + lane;
            const bool empty = at.length == 0;
            const uint32_t buf = acc_it & 1;
            const uint32_t taddr = tmem_base + buf * BN + (static_cast<uint32_t>(quadrant * 32) << 16);
            if (!empty) {
                mbar_wait(&ctl->tmem_full[buf], (acc_it >> 1) & 1, wait_ctx, 0x400 | buf);
                tcgen05_fence_after_sync();
            }
#pragma unroll 1
            for (int col = 32 * half; col < BN && at.n0 + col < p.n && row0 < p.m; col += 64) {
                uint32_t acc[32] = {};
                __syncwarp();
                if (!empty) {
                    tmem_ld_32x32(taddr + col, acc);
                    tmem_wait_ld();
                }
                if (p.out_vec) {
                    // a box in the 64-byte swizzle; its store clips rows and columns outside the gradient
                    uint8_t *const box = boxes + ((warp - 2) * 2 + (box_it++ & 1)) * OUT_BOX_BYTES;
                    if (lane == 0) tma_store_wait_read<1>();  // the box of two steps ago has been read
                    __syncwarp();
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        uint4 packed;
                        packed.x = pack2(__uint_as_float(acc[v * 8 + 0]), __uint_as_float(acc[v * 8 + 1]), bf16);
                        packed.y = pack2(__uint_as_float(acc[v * 8 + 2]), __uint_as_float(acc[v * 8 + 3]), bf16);
                        packed.z = pack2(__uint_as_float(acc[v * 8 + 4]), __uint_as_float(acc[v * 8 + 5]), bf16);
                        packed.w = pack2(__uint_as_float(acc[v * 8 + 6]), __uint_as_float(acc[v * 8 + 7]), bf16);
                        *reinterpret_cast<uint4 *>(box + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)) = packed;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&map_out, box, at.n0 + col, row0, at.run);
                        tma_store_commit();
                    }
                } else if (row < p.m) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (at.n0 + col + j < p.n)
                            store16(p.out, at.run * p.out_batch_stride + row * p.out_stride0 + (at.n0 + col + j) * p.out_stride1,
                                    __uint_as_float(acc[j]), bf16);
                }
            }
            if (!empty) {
                tcgen05_fence_before_sync();
                if (CG == 1 || leader) mbar_arrive(&ctl->tmem_empty[buf]);
                else mbar_arrive_cluster(&ctl->tmem_empty[buf], 0);
                ++acc_it;
            }
        }
        if (lane == 0) tma_store_wait<0>();
    }

    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc<CG>(tmem_base, TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------
// Plain kernels for operands that no tensor map can address: one thread per output element, fp32 sums, one rounding.
// ---------------------------------------------------------------------------
constexpr int PLAIN_ROWS = 8;

// low (may be nullptr, as may adapters): fp32 [rows, rank], added as low . up of the run's adapter.
__global__ void __launch_bounds__(256)
    grouped_plain_kernel(const Offsets offsets, const void *adapters, int64_t adapters_stride, int adapters_wide,
                         int matrices, int shared_matrix, View a, View b, const float *low, int rank, View up, int rows,
                         int n, int k, const float *scales, int64_t scales_stride, float *low_out, void *out,
                         int64_t os0, int64_t os1, int bf16) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * PLAIN_ROWS + threadIdx.x / 32;  // one warp a row
    const int run = row < rows ? run_of(offsets, rows, static_cast<int>(row)) : -1;
    if (run < 0) return;
    int matrix = run;
    if (adapters != nullptr) {
        matrix = load_index(adapters, adapters_stride, adapters_wide, run, -1, matrices);
        if (matrix >= matrices) matrix = -1;
    }
    const bool has_matrix = matrix >= 0;
    if (!shared_matrix && !has_matrix) return;
    const int64_t b_at = shared_matrix ? 0 : matrix * b.stride[0];
    for (int64_t col = static_cast<int64_t>(blockIdx.y) * 32 + (threadIdx.x & 31); col < n; col += static_cast<int64_t>(gridDim.y) * 32) {
        float acc = 0.f;
        for (int i = 0; i < k; ++i)
            acc = fmaf(load16(a.data, row * a.stride[1] + i * a.stride[2], bf16),
                       load16(b.data, b_at + i * b.stride[1] + col * b.stride[2], bf16), acc);
        if (low_out != nullptr) {
            low_out[row * n + col] = acc * scales[matrix * scales_stride];
            continue;
        }
        if (low != nullptr && has_matrix)
            for (int i = 0; i < rank; ++i)
                acc = fmaf(low[row * rank + i], load16(up.data, matrix * up.stride[0] + i * up.stride[1] + col * up.stride[2], bf16), acc);
        store16(out, row * os0 + col * os1, acc, bf16);
    }
}

__global__ void __launch_bounds__(256)
    grouped_grad_plain_kernel(const Offsets offsets, View a, View b, int rows, int m, int n, void *out, int64_t ob,
                              int64_t os0, int64_t os1, int bf16) {
    __shared__ int bounds[2];
    const int run = blockIdx.z;
    if (threadIdx.x == 0) {
        int begin = 0, end = 0;
        for (int e = 0; e <= run + 1; ++e) {
            begin = end;
            end = max(end, load_index(offsets.data, offsets.stride, offsets.wide, e, 0, rows));
        }
        bounds[0] = begin;
        bounds[1] = end;
    }
    __syncthreads();
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * PLAIN_ROWS + threadIdx.x / 32; row < m; row += static_cast<int64_t>(gridDim.x) * PLAIN_ROWS)
        for (int64_t col = static_cast<int64_t>(blockIdx.y) * 32 + (threadIdx.x & 31); col < n; col += static_cast<int64_t>(gridDim.y) * 32) {
            float acc = 0.f;
            for (int64_t t = bounds[0]; t < bounds[1]; ++t)
                acc = fmaf(load16(a.data, t * a.stride[1] + row * a.stride[2], bf16),
                           load16(b.data, t * b.stride[1] + col * b.stride[2], bf16), acc);
            store16(out, run * ob + row * os0 + col * os1, acc, bf16);
        }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Rows with unit stride and 16-byte aligned starts.  A dimension of one element has no stride of its own.
bool rows_addressable(const void *data, int64_t rows, int64_t cols, int64_t stride0, int64_t stride1) {
    return aligned16(data) && cols > 0 && (stride1 == 1 || cols == 1) &&
           (rows <= 1 || (stride0 % 8 == 0 && stride0 >= cols && stride0 < (1LL << 38)));
}

int64_t row_pitch(int64_t rows, int64_t cols, int64_t stride0) { return rows <= 1 ? (cols + 7) / 8 * 8 : stride0; }

// Matrices [count, rows, cols]: which of the last two dimensions is the unit-stride one, and whether a three-dimensional
// tensor map can address them.
struct Matrices {
    const void *data;
    int64_t count, rows, cols, stride0, stride1, stride2;
    bool mn() const { return rows_addressable(data, rows, cols, stride1, stride2); }
    bool k_major() const { return rows_addressable(data, cols, rows, stride2, stride1); }
    // (matrices need not lie one behind the other: a weight held as [rows, count, cols] has its matrices between each other's rows)
    bool batch_ok() const { return count <= 1 || (stride0 % 8 == 0 && stride0 > 0 && stride0 < (1LL << 38)); }
    bool addressable() const { return (mn() || k_major()) && batch_ok(); }
    bool use_mn() const { return mn() && batch_ok(); }
};

int map_rows(const DeviceState &dev, CUtensorMap *map, int dtype, const void *data, int64_t rows, int64_t cols,
             int64_t stride0, uint32_t box_cols, uint32_t box_rows) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(row_pitch(rows, cols, stride0)) * 2};
    const uint32_t box[2] = {box_cols, box_rows};
    return make_tensor_map(dev, map, dtype, 2, data, dims, strides, box, true);
}

// 32-bit sums, a row's in whole blocks of RANK_BLOCK.
int map_sums(const DeviceState &dev, CUtensorMap *map, const void *data, int64_t rows, int64_t pitch, uint32_t box_rows) {
    const uint64_t dims[2] = {static_cast<uint64_t>(pitch), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(pitch) * 4};
    const uint32_t box[2] = {RANK_BLOCK, box_rows};
    return make_tensor_map(dev, map, NINETOOTHED_FLOAT32, 2, data, dims, strides, box, true);
}

// box_inner x box_outer boxes over one matrix at a time
int map_matrices(const DeviceState &dev, CUtensorMap *map, int dtype, const Matrices &t, bool mn, uint32_t box_inner,
                 uint32_t box_outer) {
    const int64_t inner = mn ? t.cols : t.rows, outer = mn ? t.rows : t.cols;
    const int64_t pitch = row_pitch(outer, inner, mn ? t.stride1 : t.stride2);
    const int64_t batch = t.count <= 1 ? pitch * outer : t.stride0;
    const uint64_t dims[3] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(outer), static_cast<uint64_t>(t.count)};
    const uint64_t strides[2] = {static_cast<uint64_t>(pitch) * 2, static_cast<uint64_t>(batch) * 2};
    const uint32_t box[3] = {box_inner, box_outer, 1};
    return make_tensor_map(dev, map, dtype, 3, t.data, dims, strides, box, true);
}

// 32 x 32 boxes of row-major matrices, in the 64-byte swizzle (for stores).
int map_boxes(const DeviceState &dev, CUtensorMap *map, int dtype, const Matrices &t) {
    const int64_t pitch = row_pitch(t.rows, t.cols, t.stride1), batch = t.count <= 1 ? pitch * t.rows : t.stride0;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(t.cols), static_cast<cuuint64_t>(t.rows), static_cast<cuuint64_t>(t.count)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch) * 2, static_cast<cuuint64_t>(batch) * 2};
    const cuuint32_t box[3] = {32, 32, 1}, ones[3] = {1, 1, 1};
    const CUresult rc = dev.encode_tiled(
        map, dtype == NINETOOTHED_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
        const_cast<void *>(t.data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS)
        return fail(NINETOOTHED_B200_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the output (CUresult %d): base %p dims [%lld %lld %lld]",
                    static_cast<int>(rc), t.data, (long long)t.cols, (long long)t.rows, (long long)t.count);
    return 0;
}

template <typename Kernel>
int active_pairs(Kernel kernel, const DeviceState &dev, int threads) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(dev.sm_count / 2 * 2));
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = MAX_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {2, 1, 1};
    config.attrs = attr;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        return 0;
    }
    return clusters;
}

struct LoraMaps {
    CUtensorMap w, x, x32, x16, low, up;
};

template <int CG, int NT, bool W_MN, bool WIDE>
int launch_lora_kernel(cudaStream_t stream, const DeviceState &dev, const LoraMaps &maps, const Params &p, int64_t most_tiles) {
    auto kernel = lora_kernel<CG, NT, W_MN, WIDE>;
    static_assert(turned_smem<CG, NT, false, false>(MAX_RUNS) <= MAX_SMEM, "shared memory per CTA");
    static thread_local int configured_device = -1;
    static thread_local int pairs = 0;
    if (configured_device != dev.device) {
        NT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MAX_SMEM)));
        if constexpr (CG == 2) pairs = active_pairs(kernel, dev, lora_threads(WIDE));
        configured_device = dev.device;
    }
    const int workers = CG == 2 ? pairs : dev.sm_count;
    if (workers <= 0) return fail(NINETOOTHED_B200_ERR_DEVICE, "lora_matmul: no CTA pair fits this device");
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(most_tiles, workers) * CG));
    config.blockDim = dim3(lora_threads(WIDE));
    config.dynamicSmemBytes = turned_smem<CG, NT, false, false>(p.offsets.runs);
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    config.attrs = attr;
    config.numAttrs = 0;
    if (CG == 2) {
        attr[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[config.numAttrs++].val.clusterDim = {2, 1, 1};
    }
    if (p.matrices > 0) {  // starts under the kernel that computes scales (lhs . down)
        attr[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    NT_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, maps.w, maps.x, maps.x32, maps.x16, maps.low, maps.up, p));
    return 0;
}

// Tensor maps, then the launch.  up and low: null where there are no adapters.
template <int CG, int NT, bool WIDE>
int launch_lora(cudaStream_t stream, const DeviceState &dev, int dtype, Params &p, const void *lhs, int64_t lhs_stride0,
                const Matrices &rhs, const Matrices *up, const void *low) {
    using S = Turned<CG, NT>;
    p.n_tiles = static_cast<int>((static_cast<int64_t>(p.n) + S::TILE_N - 1) / S::TILE_N);
    p.k_blocks = (p.k + S::DEPTH - 1) / S::DEPTH;
    p.group_m = std::max(1, 2048 / NT);
    const bool mn = rhs.use_mn();
    LoraMaps maps;
    if (int rc = map_matrices(dev, &maps.w, dtype, rhs, mn, 64, mn ? S::DEPTH : BM)) return rc;
    if (int rc = map_rows(dev, &maps.x, dtype, lhs, p.rows, p.k, lhs_stride0, BK, S::ROWS_CTA)) return rc;
    if (int rc = map_rows(dev, &maps.x32, dtype, lhs, p.rows, p.k, lhs_stride0, BK, 32)) return rc;
    if (int rc = map_rows(dev, &maps.x16, dtype, lhs, p.rows, p.k, lhs_stride0, BK, 16)) return rc;
    maps.up = maps.low = maps.x;
    if (up != nullptr) {
        p.up_mn = up->use_mn();
        const int64_t pitch = p.rank_blocks * RANK_BLOCK;
        if (int rc = map_matrices(dev, &maps.up, dtype, *up, p.up_mn, 64, p.up_mn ? RANK_BLOCK : BM)) return rc;
        if (int rc = WIDE ? map_sums(dev, &maps.low, low, p.rows, pitch, S::ROWS_CTA)
                          : map_rows(dev, &maps.low, dtype, low, p.rows, 2 * pitch, 2 * pitch, BK, S::ROWS_CTA))
            return rc;
    }
    const int64_t columns = p.rows + (16 * CG - 1) * static_cast<int64_t>(std::min(p.offsets.runs, p.rows));
    const int64_t most = (columns + NT - 1) / NT * p.n_tiles;
    if (most > INT_MAX / 16) return fail(NINETOOTHED_B200_ERR_SHAPE, "lora_matmul: too many tiles");
    return mn ? launch_lora_kernel<CG, NT, true, WIDE>(stream, dev, maps, p, most) : launch_lora_kernel<CG, NT, false, WIDE>(stream, dev, maps, p, most);
}

template <int CG, int NT, bool W_MN, bool SPLIT, Job JOB>
int launch_turned_kernel(cudaStream_t stream, const DeviceState &dev, const CUtensorMap &map_w, const CUtensorMap &map_x,
                         const CUtensorMap &map_x_chunk, const Params &p, int64_t most_tiles) {
    auto kernel = turned_kernel<CG, NT, W_MN, SPLIT, JOB>;
    static_assert(turned_smem<CG, NT, SPLIT, JOB == JOB_FEW>(MAX_RUNS) <= MAX_SMEM, "shared memory per CTA");
    static thread_local int configured_device = -1;
    static thread_local int pairs = 0;
    if (configured_device != dev.device) {
        NT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MAX_SMEM)));
        if constexpr (CG == 2) pairs = active_pairs(kernel, dev, NUM_THREADS);
        configured_device = dev.device;
    }
    cudaLaunchConfig_t config = {};
    const int64_t workers = SPLIT ? most_tiles : std::min<int64_t>(most_tiles, CG == 2 ? pairs : dev.sm_count);
    if (workers <= 0) return fail(NINETOOTHED_B200_ERR_DEVICE, "grouped matmul: no CTA pair fits this device");
    const int cluster = SPLIT ? p.split : CG;
    config.gridDim = dim3(static_cast<unsigned>(workers * cluster));
    config.blockDim = dim3(NUM_THREADS);
    config.dynamicSmemBytes = turned_smem<CG, NT, SPLIT, JOB == JOB_FEW>(p.offsets.runs);
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    config.attrs = attr;
    config.numAttrs = 0;
    if (cluster > 1) {
        attr[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[config.numAttrs++].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    }
    if (JOB == JOB_FEW && p.low_chunks > 0) {  // starts under the kernel before it
        attr[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    NT_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, map_w, map_x, map_x_chunk, p));
    return 0;
}

template <int CG, int NT, bool SPLIT, Job JOB>
int launch_turned(cudaStream_t stream, const DeviceState &dev, int dtype, Params &p, const void *lhs, int64_t lhs_stride0,
                  const Matrices &rhs, int64_t live_runs) {
    using S = Turned<CG, NT>;
    p.n_tiles = static_cast<int>((static_cast<int64_t>(p.n) + S::TILE_N - 1) / S::TILE_N);
    p.k_blocks = (p.k + S::DEPTH - 1) / S::DEPTH;
    p.group_m = std::max(1, 2048 / NT);
    const bool mn = rhs.use_mn();
    CUtensorMap map_w, map_x, map_x_chunk;
    if (int rc = map_matrices(dev, &map_w, dtype, rhs, mn, 64, mn ? S::DEPTH : BM)) return rc;
    if (int rc = map_rows(dev, &map_x, dtype, lhs, p.rows, p.k, lhs_stride0, BK, S::ROWS_CTA)) return rc;
    if (int rc = map_rows(dev, &map_x_chunk, dtype, lhs, p.rows, p.k, lhs_stride0, BK, A_CHUNK_ROWS)) return rc;
    const int64_t most = (JOB == JOB_FEW ? (p.rows + NT - 1) / NT : live_runs + p.rows / NT) * p.n_tiles;
    if (most > INT_MAX / 16) return fail(NINETOOTHED_B200_ERR_SHAPE, "grouped matmul: too many tiles");
    return mn ? launch_turned_kernel<CG, NT, true, SPLIT, JOB>(stream, dev, map_w, map_x, map_x_chunk, p, most)
              : launch_turned_kernel<CG, NT, false, SPLIT, JOB>(stream, dev, map_w, map_x, map_x_chunk, p, most);
}

// Which tiles a grouped product gets.  The bounds lie on the device, so the host goes by averages: `live` runs at most
// hold rows, and a run of r rows makes about r / NT + 1/2 tiles.
//   - Fewer tiles than half the SMs: clusters of 2 to 8 CTAs share each tile's reduction (one row against two 4096 x 2048
//     matrices: 16.0 us without, 11.2 with four CTAs a tile).
//   - Otherwise the width with the least modelled time, waves x blocks x cycles per 128-deep block (830 for 64 rows, 1080
//     for 128, 1400 for 256 on a pair: between the 1540 measured where all SMs wait for memory and the 1100 of the products).
//     Runs of 96, 192 and 384 rows against eight 4096 x 1024 matrices take 19.7, 30.5, 42.5 us with 64 rows a tile, 23.3,
//     24.3, 39.4 with 128, 24.2, 30.3, 31.4 with 256; 29 runs of 172 rows on average against 1544 x 1160 ones 58, 45, 39.
int launch_grouped(cudaStream_t stream, const DeviceState &dev, int dtype, Params &p, const void *lhs, int64_t lhs_stride0,
                   const Matrices &rhs, int64_t live) {
    const int64_t n_tiles = (static_cast<int64_t>(p.n) + BM - 1) / BM;
    const int64_t few = (live + p.rows / SPLIT_NT) * n_tiles, blocks = (static_cast<int64_t>(p.k) + 2 * BK - 1) / (2 * BK);
    p.split = 1;
    while (p.split < 8 && few * p.split * 2 <= dev.sm_count && blocks >= p.split * 4) p.split *= 2;
    if (p.split > 1) return launch_turned<1, SPLIT_NT, true, JOB_PRODUCT>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, live);
    const auto cost = [&](int64_t rows, int64_t columns, int64_t workers, int64_t cycles) {
        const int64_t halves = std::max<int64_t>(2 * live, 2 * p.rows / rows + live);  // half tiles
        const int64_t tiles = (halves * ((p.n + columns - 1) / columns) + 1) / 2;
        return (tiles + workers - 1) / workers * cycles;
    };
    const int64_t narrow = cost(64, 128, dev.sm_count, 830), middle = cost(128, 128, dev.sm_count, 1080),
                  wide = cost(256, 256, dev.sm_count / 2, 1400);
    if (narrow <= middle && narrow <= wide)
        return launch_turned<1, 64, false, JOB_PRODUCT>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, live);
    if (middle <= wide) return launch_turned<1, 128, false, JOB_PRODUCT>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, live);
    return launch_turned<2, 256, false, JOB_PRODUCT>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, live);
}

int64_t low_chunks(int64_t k) { return (k + LOW_CHUNK - 1) / LOW_CHUNK; }

// Few rows, or requests of few rows each: the adapters' part costs no tile of its own and runs under the streaming of rhs, a row
// at a time, which takes about 5.5 ns x (rank + 22) a row.  Otherwise a request takes at least 16 columns of a tile, whatever its
// rows, which is 0.8 us a request, 145 of those units.  The constant behind them is what the launch before the projection takes
// more where it goes by tiles, 3600 units, or, where k is short beside the rank, what is missing of a streaming to run under.  All
// three are fitted to these times in us, this way / the other (rows in requests, bf16):
//   4096 x 4096, rank 16: 16 in 1 16 / 24, 64 in 64 21 / 63, 64 in 4 20 / 27, 256 in 64 48 / 64, 256 in 16 48 / 32,
//   512 in 128 96 / 116, 512 in 64 96 / 65, 2048 in 2048 488 / 1623, 6000 in 2048 1394 / 1669, 8192 in 2048 1895 / 1661
//   4096 x 4096, rank 8: 128 in 4 23 / 29, 256 in 4 43 / 28, 256 in 64 44 / 65
//   4096 x 1024, rank 8: 2048 in 2048 166 / 654, 8192 in 2048 576 / 681
//   4096 x 4096, rank 64: 1 in 1 19 / 25, 16 in 4 22 / 29, 64 in 64 39 / 73, 64 in 4 36 / 29, 1024 in 512 466 / 465
//   1024 x 2048, rank 64: 1 in 1 21 / 12, 64 in 64 34 / 28, 128 in 128 32 / 44, 128 in 32 34 / 26, 512 in 256 88 / 86
// (fp16 takes as long this way and 2 to 45 % longer the other, most for ranks that are much beside k.)
bool few_rows(int64_t rows, int64_t k, int64_t rank, int64_t requests) {
    return rank <= FEW_RANK && rows * (rank + 22) < requests * 145 + (k >= 32 * rank ? 3600 : -4000);
}

size_t lora_workspace(int64_t rows, int64_t k, int64_t rank) {
    const size_t parts = static_cast<size_t>(rows) * ((rank + RANK_BLOCK - 1) / RANK_BLOCK) * RANK_BLOCK * 4;
    const size_t sums = few_rows(rows, k, rank, std::min<int64_t>(rows, MAX_RUNS)) ? static_cast<size_t>(low_chunks(k)) * rows * rank * 4 : 0;
    return std::max(parts, sums);
}

int launch_few(cudaStream_t stream, const DeviceState &dev, int dtype, Params &p, const void *lhs, int64_t lhs_stride0,
               const Matrices &rhs, const Matrices &down, const Matrices &up, float *low) {
    p.low_chunks = 0;
    if (p.matrices > 0) {
        p.low = low;
        p.low_chunks = static_cast<int>(low_chunks(p.k));
        p.up = up.data;
        p.up_mn = up.use_mn();
        p.up_stride[0] = up.stride0;
        p.up_stride[1] = up.stride1;
        p.up_stride[2] = up.stride2;
        const int64_t tasks = static_cast<int64_t>(p.rows) * p.low_chunks * ((p.rank + 7) / 8);
        low_kernel<<<static_cast<unsigned>(tasks), LOW_WARPS * 32, 0, stream>>>(
            p, lhs, lhs_stride0, View{down.data, {down.stride0, down.stride1, down.stride2}}, down.use_mn(), low);
        NT_CUDA_CHECK(cudaGetLastError());
    }
    const int64_t tiles = (static_cast<int64_t>(p.rows) + SPLIT_NT - 1) / SPLIT_NT * ((static_cast<int64_t>(p.n) + BM - 1) / BM);
    const int64_t blocks = (static_cast<int64_t>(p.k) + 2 * BK - 1) / (2 * BK);
    p.split = 1;
    while (p.split < 8 && tiles * p.split * 2 <= dev.sm_count && blocks >= p.split * 2) p.split *= 2;
    return launch_turned<1, SPLIT_NT, true, JOB_FEW>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, 1);
}

bool has_arrays(const NineToothedTensor &t) { return t.shape != nullptr && t.strides != nullptr; }

constexpr int64_t MAX_DIM = INT_MAX - 65536;  // coordinates of a tile that overhangs, and padded rows, stay 32-bit

int check_offsets(const char *what, const NineToothedTensor &offsets, int64_t runs, int offsets_dtype, Offsets *out) {
    if (offsets_dtype != NINETOOTHED_INT32 && offsets_dtype != NINETOOTHED_INT64)
        return fail(NINETOOTHED_B200_ERR_DTYPE, "%s: offsets must be int32 or int64, got dtype %d", what, offsets_dtype);
    if (static_cast<int64_t>(offsets.shape[0]) != runs + 1)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: offsets must hold %lld bounds (runs + 1), got %llu", what,
                    (long long)(runs + 1), (unsigned long long)offsets.shape[0]);
    if (runs > MAX_RUNS)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: %lld runs of rows, at most %d are supported", what, (long long)runs, MAX_RUNS);
    if (!offsets.data) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null offsets", what);
    *out = Offsets{offsets.data, offsets.strides[0], offsets_dtype == NINETOOTHED_INT64 ? 1 : 0, static_cast<int>(runs)};
    return 0;
}

dim3 plain_grid(int64_t rows, int64_t cols, int64_t runs = 1) {
    return dim3(static_cast<unsigned>((rows + PLAIN_ROWS - 1) / PLAIN_ROWS),
                static_cast<unsigned>(std::min<int64_t>((cols + 31) / 32, 65535)), static_cast<unsigned>(runs));
}

// Rows of output take 16-byte stores.
bool output_vec(const NineToothedTensor &t) {
    return t.strides[1] == 1 && (t.shape[0] <= 1 || t.strides[0] % 8 == 0) && aligned16(t.data);
}

int run_grouped(cudaStream_t stream, const NineToothedTensor &lhs, const NineToothedTensor &rhs,
                const NineToothedTensor &offsets, const NineToothedTensor &output, int dtype, int offsets_dtype) {
    const char *what = "grouped_matmul";
    clear_error();
    for (auto *t : {&lhs, &rhs, &offsets, &output})
        if (!has_arrays(*t)) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null shape/strides", what);
    if (!is_16bit_float(dtype)) return fail(NINETOOTHED_B200_ERR_DTYPE, "%s: dtype %d is not fp16/bf16", what, dtype);
    const int64_t rows = lhs.shape[0], k = lhs.shape[1], runs = rhs.shape[0], n = rhs.shape[2];
    if (static_cast<int64_t>(rhs.shape[1]) != k || static_cast<int64_t>(output.shape[0]) != rows ||
        static_cast<int64_t>(output.shape[1]) != n)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: shapes do not agree (lhs [%lld, %lld], rhs [%lld, %llu, %lld], output "
                    "[%llu, %llu])", what, (long long)rows, (long long)k, (long long)runs, (unsigned long long)rhs.shape[1],
                    (long long)n, (unsigned long long)output.shape[0], (unsigned long long)output.shape[1]);
    Params p = {};
    if (int rc = check_offsets(what, offsets, runs, offsets_dtype, &p.offsets)) return rc;
    if (rows > MAX_DIM || n > MAX_DIM || k > MAX_DIM) return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: a dimension exceeds 32-bit indexing", what);
    if (rows == 0 || n == 0 || runs == 0) return 0;
    if (!output.data || (k > 0 && (!lhs.data || !rhs.data))) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null data pointer", what);
    const DeviceState *dev = nullptr;
    if (int rc = current_device_state(&dev)) return rc;
    p.matrices = static_cast<int>(runs);
    p.rows = static_cast<int>(rows);
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.k_blocks = static_cast<int>((k + BK - 1) / BK);
    p.bf16 = dtype == NINETOOTHED_BFLOAT16;
    p.out = output.data;
    p.out_stride0 = output.strides[0];
    p.out_stride1 = output.strides[1];
    p.out_vec = output_vec(output);
    p.status = dev->status;
    const Matrices matrices{rhs.data, runs, k, n, rhs.strides[0], rhs.strides[1], rhs.strides[2]};
    if (rows_addressable(lhs.data, rows, k, lhs.strides[0], lhs.strides[1]) && matrices.addressable()) {
        return launch_grouped(stream, *dev, dtype, p, lhs.data, lhs.strides[0], matrices, std::min(runs, rows));
    }
    note_plain_launch("grouped_matmul %lld x %lld x %lld runs on the plain CUDA-core kernel: the tensor-core path needs a "
                      "unit-stride K in lhs, a unit-stride dimension in every matrix of rhs, the other strides multiples "
                      "of 8 elements and 16-byte aligned bases", (long long)rows, (long long)n, (long long)k);
    grouped_plain_kernel<<<plain_grid(rows, n), 256, 0, stream>>>(
        p.offsets, nullptr, 0, 0, p.matrices, 0, View{lhs.data, {0, lhs.strides[0], lhs.strides[1]}},
        View{rhs.data, {rhs.strides[0], rhs.strides[1], rhs.strides[2]}}, nullptr, 0, View{}, p.rows, p.n, p.k, nullptr, 0,
        nullptr, output.data, output.strides[0], output.strides[1], p.bf16);
    NT_CUDA_CHECK(cudaGetLastError());
    return 0;
}

template <int CG, int BN>
int launch_grad(cudaStream_t stream, const DeviceState &dev, int dtype, const NineToothedTensor &lhs, const NineToothedTensor &grad,
                const NineToothedTensor &rhs_grad, GradParams &p) {
    auto kernel = grad_kernel<CG, BN>;
    static_assert(grad_smem<CG, BN>(MAX_RUNS) <= MAX_SMEM, "shared memory per CTA");
    static thread_local int configured_device = -1;
    static thread_local int pairs = 0;
    if (configured_device != dev.device) {
        NT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MAX_SMEM)));
        if constexpr (CG == 2) pairs = active_pairs(kernel, dev, GRAD_THREADS);
        configured_device = dev.device;
    }
    using S = Grad<CG, BN>;
    p.m_tiles = (p.m + S::TILE_M - 1) / S::TILE_M;
    p.n_tiles = (p.n + BN - 1) / BN;
    const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.offsets.runs;
    const int64_t workers = std::min<int64_t>(tiles, CG == 2 ? pairs : dev.sm_count);
    if (tiles > INT_MAX / 2) return fail(NINETOOTHED_B200_ERR_SHAPE, "grouped_matmul_rhs_grad: too many tiles");
    if (workers <= 0) return fail(NINETOOTHED_B200_ERR_DEVICE, "grouped_matmul_rhs_grad: no CTA pair fits this device");
    CUtensorMap map_a, map_b, map_out;
    if (int rc = map_rows(dev, &map_a, dtype, lhs.data, p.rows, p.m, lhs.strides[0], 64, BK)) return rc;
    if (int rc = map_rows(dev, &map_b, dtype, grad.data, p.rows, p.n, grad.strides[0], 64, BK)) return rc;
    map_out = map_a;
    const Matrices out{rhs_grad.data, p.offsets.runs, p.m, p.n, rhs_grad.strides[0], rhs_grad.strides[1], rhs_grad.strides[2]};
    p.out_vec = out.use_mn();
    if (p.out_vec)
        if (int rc = map_boxes(dev, &map_out, dtype, out)) return rc;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(workers * CG));
    config.blockDim = dim3(GRAD_THREADS);
    config.dynamicSmemBytes = grad_smem<CG, BN>(p.offsets.runs);
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    if (CG == 2) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {2, 1, 1};
        config.attrs = attr;
        config.numAttrs = 1;
    }
    NT_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, map_a, map_b, map_out, p));
    return 0;
}

int run_grouped_grad(cudaStream_t stream, const NineToothedTensor &lhs, const NineToothedTensor &grad,
                     const NineToothedTensor &offsets, const NineToothedTensor &rhs_grad, int dtype, int offsets_dtype) {
    const char *what = "grouped_matmul_rhs_grad";
    clear_error();
    for (auto *t : {&lhs, &grad, &offsets, &rhs_grad})
        if (!has_arrays(*t)) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null shape/strides", what);
    if (!is_16bit_float(dtype)) return fail(NINETOOTHED_B200_ERR_DTYPE, "%s: dtype %d is not fp16/bf16", what, dtype);
    const int64_t rows = lhs.shape[0], m = lhs.shape[1], n = grad.shape[1], runs = rhs_grad.shape[0];
    if (static_cast<int64_t>(grad.shape[0]) != rows || static_cast<int64_t>(rhs_grad.shape[1]) != m ||
        static_cast<int64_t>(rhs_grad.shape[2]) != n)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: shapes do not agree (lhs [%lld, %lld], output_grad [%llu, %lld], rhs_grad "
                    "[%lld, %llu, %llu])", what, (long long)rows, (long long)m, (unsigned long long)grad.shape[0], (long long)n,
                    (long long)runs, (unsigned long long)rhs_grad.shape[1], (unsigned long long)rhs_grad.shape[2]);
    GradParams p = {};
    if (int rc = check_offsets(what, offsets, runs, offsets_dtype, &p.offsets)) return rc;
    if (rows > MAX_DIM || n > MAX_DIM || m > MAX_DIM) return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: a dimension exceeds 32-bit indexing", what);
    if (m == 0 || n == 0 || runs == 0) return 0;
    if (!rhs_grad.data || (rows > 0 && (!lhs.data || !grad.data))) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null data pointer", what);
    const DeviceState *dev = nullptr;
    if (int rc = current_device_state(&dev)) return rc;
    p.rows = static_cast<int>(rows);
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.bf16 = dtype == NINETOOTHED_BFLOAT16;
    p.out = rhs_grad.data;
    p.out_batch_stride = rhs_grad.strides[0];
    p.out_stride0 = rhs_grad.strides[1];
    p.out_stride1 = rhs_grad.strides[2];
    p.status = dev->status;
    if (rows > 0 && rows_addressable(lhs.data, rows, m, lhs.strides[0], lhs.strides[1]) &&
        rows_addressable(grad.data, rows, n, grad.strides[0], grad.strides[1])) {
        const int64_t wide = runs * ((m + 255) / 256) * ((n + 255) / 256);
        return wide * 2 >= dev->sm_count ? launch_grad<2, 256>(stream, *dev, dtype, lhs, grad, rhs_grad, p)
                                         : launch_grad<1, 128>(stream, *dev, dtype, lhs, grad, rhs_grad, p);
    }
    if (rows > 0)
        note_plain_launch("grouped_matmul_rhs_grad %lld x %lld x %lld runs on the plain CUDA-core kernel: the tensor-core path "
                          "needs unit-stride columns, row strides that are multiples of 8 elements and 16-byte aligned bases",
                          (long long)rows, (long long)m, (long long)n);
    dim3 grid = plain_grid(m, n, runs);
    grouped_grad_plain_kernel<<<grid, 256, 0, stream>>>(p.offsets, View{lhs.data, {0, lhs.strides[0], lhs.strides[1]}},
                                                        View{grad.data, {0, grad.strides[0], grad.strides[1]}}, p.rows, p.m,
                                                        p.n, rhs_grad.data, rhs_grad.strides[0], rhs_grad.strides[1],
                                                        rhs_grad.strides[2], p.bf16);
    NT_CUDA_CHECK(cudaGetLastError());
    return 0;
}

// Many rows under adapters: first scales (lhs . down), then the projection with the second products.
int launch_many(cudaStream_t stream, const DeviceState &dev, int dtype, Params &p, const void *lhs, int64_t lhs_stride0,
                const Matrices &rhs, const Matrices &down, const Matrices &up, void *workspace) {
    const bool any = p.matrices > 0;
    if (any) {
        Params parts = p;
        parts.n = p.rank;
        parts.out = workspace;
        parts.out_stride0 = p.rank_blocks * RANK_BLOCK;
        parts.out_stride1 = 1;
        const int64_t live = std::min(p.offsets.runs, p.rows), n_tiles = (p.rank + BM - 1) / BM;
        const int64_t blocks = (static_cast<int64_t>(p.k) + 2 * BK - 1) / (2 * BK), narrow = (live + p.rows / 64) * n_tiles;
        parts.split = 1;
        while (parts.split < 8 && narrow * parts.split * 2 <= dev.sm_count && blocks >= parts.split * 2) parts.split *= 2;
        int rc;
        if (parts.split > 1) rc = launch_turned<1, SPLIT_NT, true, JOB_PARTS>(stream, dev, dtype, parts, lhs, lhs_stride0, down, live);
        else if (narrow <= 2 * dev.sm_count) rc = launch_turned<1, 64, false, JOB_PARTS>(stream, dev, dtype, parts, lhs, lhs_stride0, down, live);
        else rc = launch_turned<1, 128, false, JOB_PARTS>(stream, dev, dtype, parts, lhs, lhs_stride0, down, live);
        if (rc != 0) return rc;
    }
    // Tiles of 256 x 256 on CTA pairs, or 128 x 128 on single CTAs where that takes fewer waves' time (as in launch_grouped).
    // A request's columns are padded to steps of 16, of 32 on a pair: by half a step, taken over all.
    const auto waves = [&](int64_t width, int64_t step, int64_t workers) {
        const int64_t columns = p.rows + step / 2 * static_cast<int64_t>(std::min(p.offsets.runs, p.rows));
        return ((columns + width - 1) / width * ((p.n + width - 1) / width) + workers - 1) / workers;
    };
    if (1400 * waves(256, 32, dev.sm_count / 2) <= 1080 * waves(128, 16, dev.sm_count))
        return p.bf16 ? launch_lora<2, 256, false>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, any ? &up : nullptr, workspace)
                      : launch_lora<2, 256, true>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, any ? &up : nullptr, workspace);
    return p.bf16 ? launch_lora<1, 128, false>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, any ? &up : nullptr, workspace)
                  : launch_lora<1, 128, true>(stream, dev, dtype, p, lhs, lhs_stride0, rhs, any ? &up : nullptr, workspace);
}

int run_lora(cudaStream_t stream, const NineToothedTensor &lhs, const NineToothedTensor &rhs, const NineToothedTensor &down,
             const NineToothedTensor &up, const NineToothedTensor &scales, const NineToothedTensor &offsets,
             const NineToothedTensor &adapters, const NineToothedTensor &output, int dtype, int offsets_dtype,
             int adapters_dtype, void *workspace, size_t workspace_size) {
    const char *what = "lora_matmul";
    clear_error();
    for (auto *t : {&lhs, &rhs, &down, &up, &scales, &offsets, &adapters, &output})
        if (!has_arrays(*t)) return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null shape/strides", what);
    if (!is_16bit_float(dtype)) return fail(NINETOOTHED_B200_ERR_DTYPE, "%s: dtype %d is not fp16/bf16", what, dtype);
    const int64_t rows = lhs.shape[0], k = lhs.shape[1], n = rhs.shape[1], count = down.shape[0], rank = down.shape[2],
                  runs = adapters.shape[0];
    if (static_cast<int64_t>(rhs.shape[0]) != k || static_cast<int64_t>(down.shape[1]) != k ||
        static_cast<int64_t>(up.shape[0]) != count || static_cast<int64_t>(up.shape[1]) != rank ||
        static_cast<int64_t>(up.shape[2]) != n || static_cast<int64_t>(scales.shape[0]) != count ||
        static_cast<int64_t>(output.shape[0]) != rows || static_cast<int64_t>(output.shape[1]) != n)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: shapes do not agree (lhs [%lld, %lld], rhs [%llu, %lld], down [%lld, %llu, "
                    "%lld], up [%llu, %llu, %llu], scales [%llu], output [%llu, %llu])", what, (long long)rows, (long long)k,
                    (unsigned long long)rhs.shape[0], (long long)n, (long long)count, (unsigned long long)down.shape[1],
                    (long long)rank, (unsigned long long)up.shape[0], (unsigned long long)up.shape[1],
                    (unsigned long long)up.shape[2], (unsigned long long)scales.shape[0],
                    (unsigned long long)output.shape[0], (unsigned long long)output.shape[1]);
    if (adapters_dtype != NINETOOTHED_INT32 && adapters_dtype != NINETOOTHED_INT64)
        return fail(NINETOOTHED_B200_ERR_DTYPE, "%s: adapters must be int32 or int64, got dtype %d", what, adapters_dtype);
    Params p = {};
    if (int rc = check_offsets(what, offsets, runs, offsets_dtype, &p.offsets)) return rc;
    if (rows > MAX_DIM || n > MAX_DIM || k > MAX_DIM || rank > MAX_DIM / 2 || count > MAX_DIM)
        return fail(NINETOOTHED_B200_ERR_SHAPE, "%s: a dimension exceeds 32-bit indexing", what);
    if (rows == 0 || n == 0 || runs == 0) return 0;
    const bool any = count > 0 && rank > 0;  // there are adapters at all
    if (!output.data || !adapters.data || (k > 0 && (!lhs.data || !rhs.data)) ||
        (any && (!down.data || !up.data || !scales.data)))
        return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: null data pointer", what);
    const size_t needed = lora_workspace(rows, k, rank);
    if (any && (workspace == nullptr || workspace_size < needed || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
        return fail(NINETOOTHED_B200_ERR_ARGUMENT, "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu at %p", what,
                    needed, workspace_size, workspace);
    const DeviceState *dev = nullptr;
    if (int rc = current_device_state(&dev)) return rc;
    p.adapters = adapters.data;
    p.adapters_stride = adapters.strides[0];
    p.adapters_wide = adapters_dtype == NINETOOTHED_INT64;
    p.matrices = any ? static_cast<int>(count) : 0;
    p.rows = static_cast<int>(rows);
    p.k = static_cast<int>(k);
    p.k_blocks = static_cast<int>((k + BK - 1) / BK);
    p.bf16 = dtype == NINETOOTHED_BFLOAT16;
    p.scales = static_cast<const float *>(scales.data);
    p.scales_stride = scales.strides[0];
    // (without adapters the shapes' rank says nothing: no kernel may size or fill anything by it)
    p.rank = any ? static_cast<int>(rank) : 0;
    p.rank_blocks = (p.rank + RANK_BLOCK - 1) / RANK_BLOCK;
    p.status = dev->status;
    const Matrices shared{rhs.data, 1, k, n, 0, rhs.strides[0], rhs.strides[1]};
    const Matrices first{down.data, count, k, rank, down.strides[0], down.strides[1], down.strides[2]};
    const Matrices second{up.data, count, rank, n, up.strides[0], up.strides[1], up.strides[2]};
    if (rows_addressable(lhs.data, rows, k, lhs.strides[0], lhs.strides[1]) && shared.addressable() &&
        (!any || (first.addressable() && second.addressable()))) {
        p.n = static_cast<int>(n);
        p.out = output.data;
        p.out_stride0 = output.strides[0];
        p.out_stride1 = output.strides[1];
        p.out_vec = output_vec(output);
        if (any ? few_rows(rows, k, rank, std::min(runs, rows)) : rows <= SPLIT_NT)
            return launch_few(stream, *dev, dtype, p, lhs.data, lhs.strides[0], shared, first, second, static_cast<float *>(workspace));
        return launch_many(stream, *dev, dtype, p, lhs.data, lhs.strides[0], shared, first, second, workspace);
    }
    note_plain_launch("lora_matmul %lld x %lld x %lld, rank %lld, runs on the plain CUDA-core kernels: the tensor-core path needs "
                      "a unit-stride K in lhs, a unit-stride dimension in rhs, down and up, the other strides multiples of 8 "
                      "elements and 16-byte aligned bases", (long long)rows, (long long)n, (long long)k, (long long)rank);
    const View a{lhs.data, {0, lhs.strides[0], lhs.strides[1]}};
    const View up_view{up.data, {up.strides[0], up.strides[1], up.strides[2]}};
    float *low = static_cast<float *>(workspace);
    if (any) {
        grouped_plain_kernel<<<plain_grid(rows, rank), 256, 0, stream>>>(
            p.offsets, p.adapters, p.adapters_stride, p.adapters_wide, p.matrices, 0, a,
            View{down.data, {down.strides[0], down.strides[1], down.strides[2]}}, nullptr, 0, View{}, p.rows, p.rank, p.k,
            p.scales, p.scales_stride, low, nullptr, 0, 0, p.bf16);
        NT_CUDA_CHECK(cudaGetLastError());
    }
    grouped_plain_kernel<<<plain_grid(rows, n), 256, 0, stream>>>(
        p.offsets, p.adapters, p.adapters_stride, p.adapters_wide, p.matrices, 1, a, View{rhs.data, {0, rhs.strides[0], rhs.strides[1]}},
        any ? low : nullptr, p.rank, up_view, p.rows, static_cast<int>(n), p.k, nullptr, 0, nullptr, output.data,
        output.strides[0], output.strides[1], p.bf16);
    NT_CUDA_CHECK(cudaGetLastError());
    return 0;
}

}  // namespace
}  // namespace nt

extern "C" {

NineToothedResult launch_grouped_matmul(NineToothedStream stream, NineToothedTensor lhs, NineToothedTensor rhs,
                                        NineToothedTensor offsets, NineToothedTensor output, int dtype, int offsets_dtype) {
    return nt::run_grouped(static_cast<cudaStream_t>(stream), lhs, rhs, offsets, output, dtype, offsets_dtype);
}

NineToothedResult launch_grouped_matmul_rhs_grad(NineToothedStream stream, NineToothedTensor lhs, NineToothedTensor output_grad,
                                                 NineToothedTensor offsets, NineToothedTensor rhs_grad, int dtype,
                                                 int offsets_dtype) {
    return nt::run_grouped_grad(static_cast<cudaStream_t>(stream), lhs, output_grad, offsets, rhs_grad, dtype, offsets_dtype);
}

NineToothedResult launch_lora_matmul(NineToothedStream stream, NineToothedTensor lhs, NineToothedTensor rhs, NineToothedTensor down,
                                     NineToothedTensor up, NineToothedTensor scales, NineToothedTensor offsets,
                                     NineToothedTensor adapters, NineToothedTensor output, int dtype, int offsets_dtype,
                                     int adapters_dtype, void *workspace, size_t workspace_size) {
    return nt::run_lora(static_cast<cudaStream_t>(stream), lhs, rhs, down, up, scales, offsets, adapters, output, dtype,
                        offsets_dtype, adapters_dtype, workspace, workspace_size);
}

size_t launch_lora_matmul_workspace_size(NineToothedTensor lhs, NineToothedTensor down) {
    if (!lhs.shape || !down.shape) return 0;
    if (lhs.shape[0] > static_cast<uint64_t>(nt::MAX_DIM) || down.shape[2] > static_cast<uint64_t>(nt::MAX_DIM)) return 0;
    return nt::lora_workspace(static_cast<int64_t>(lhs.shape[0]), static_cast<int64_t>(lhs.shape[1]), static_cast<int64_t>(down.shape[2]));
}

}  // extern "C"
