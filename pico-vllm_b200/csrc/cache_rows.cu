// Rows of the cache moved inside their own tensors: pages copied to other pages, and the states of a request's beams passed on to the beams that
// come of them.  Nothing is computed: what bounds both is reading every row that is copied once and writing every row that is overwritten once.
//
// A tensor is [outer, rows, ...] with the bytes of a row in one piece; "row r" is the rows r of all its outer entries (a page of every layer, the
// state of a request in every layer).  Sizes, strides and starts may be any: 16 bytes go at a time where all of them allow it.
#include "common.cuh"
#include <atomic>

#define ROWS_TENSORS 16                                         // tensors of one launch
#define ROWS_THREADS 256
#define ROWS_LOADS 4                                            // loads of a thread under way
#define ROWS_SPAN (ROWS_THREADS * ROWS_LOADS)                   // units of a block
#define SHIFT_LOADS 2                                           // ... where words are put together
#define SHIFT_SPAN (ROWS_THREADS * SHIFT_LOADS)
#define ROWS_BEAMS 32                                           // places of a group: lanes of a warp

__device__ unsigned g_rows_missed = 0;  // how often an index outside a tensor was met (and passed over); only ever counted up
// *out: has one been met since this was asked last, on this device, by what the stream has run?  Waits for the stream and for no other: waiting for the device would end
// a recording that another thread is making.  What was told last is kept on the host and the count is never set back, so that nothing that a kernel counts
// meanwhile, or on another stream, is lost: it is told the next time.  A stream that is being recorded is not asked.
PICO_API int pico_rows_status(int* out, cudaStream_t stream) {
    static std::atomic<unsigned> told[64];
    int dev = 0;
    unsigned now = 0;
    cudaStreamCaptureStatus recording = cudaStreamCaptureStatusNone;
    *out = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64)) return PICO_ERR_SIZE;
    if (e == cudaSuccess) e = cudaStreamIsCapturing(stream, &recording);
    if (e == cudaSuccess && recording != cudaStreamCaptureStatusNone) return 0;
    if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&now, g_rows_missed, sizeof(now), 0, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) return (int)e;
    // (two threads that ask at once: one of them tells, and an older count never takes the place of a newer)
    unsigned before = told[dev].load();
    while ((int)(now - before) > 0)
        if (told[dev].compare_exchange_weak(before, now)) {
            *out = 1;
            break;
        }
    return 0;
}

struct RowTensor {
    char* base;
    long long outer_stride, row_stride, bytes;   // bytes: of a row
    unsigned units, total;               // of a row; of a row in all outer entries
    int rows, unit;                      // unit: bytes that go at a time (in copy_shifted: that every start and size is a multiple of)
    int first;                           // the first block (x) that works on this tensor
};
struct RowTensors {
    RowTensor t[ROWS_TENSORS];
    int n, rows;                         // rows: the fewest that one of them has
};

__device__ __forceinline__ int rows_tensor(const RowTensors& ts, int block) {
    int k = 0;
    while (k + 1 < ts.n && block >= ts.t[k + 1].first) ++k;
    return k;
}

__device__ __forceinline__ void copy_aligned(const RowTensor& t, int block, int src, int dst) {
    const long long from = (long long)src * t.row_stride, to = (long long)dst * t.row_stride;
    const unsigned i0 = (unsigned)block * ROWS_SPAN + threadIdx.x;
    uint4 v[ROWS_LOADS];
    long long at[ROWS_LOADS];
#pragma unroll
    for (int u = 0; u < ROWS_LOADS; ++u) {
        const unsigned i = i0 + u * ROWS_THREADS;
        if (i < t.total) {
            const unsigned o = i / t.units;
            at[u] = (long long)o * t.outer_stride + (i - o * t.units) * 16ll;
            v[u] = *reinterpret_cast<const uint4*>(t.base + at[u] + from);
        }
    }
#pragma unroll
    for (int u = 0; u < ROWS_LOADS; ++u)
        if (i0 + u * ROWS_THREADS < t.total) *reinterpret_cast<uint4*>(t.base + at[u] + to) = v[u];
}

// The same for rows that start anywhere: the bytes of row dst are stored in whole 16-byte words, cut from the two words of row src that hold them; what
// is the row's of its first and last word goes in bytes or pairs of them.  Only words that hold bytes of the row are read.  (t.units: the words
// that a row may touch.)
__device__ __forceinline__ void copy_shifted(const RowTensor& t, int block, int src, int dst) {
    const unsigned i0 = (unsigned)block * SHIFT_SPAN + threadIdx.x;
    uint4 lo[SHIFT_LOADS], hi[SHIFT_LOADS];
    char* to[SHIFT_LOADS];
    int first[SHIFT_LOADS], last[SHIFT_LOADS], shift[SHIFT_LOADS];                     // the word's bytes first .. last - 1 are the row's
#pragma unroll
    for (int u = 0; u < SHIFT_LOADS; ++u) {
        const unsigned i = i0 + u * ROWS_THREADS, o = i / t.units;
        char* row = t.base + (long long)o * t.outer_stride;
        char* d = row + (long long)dst * t.row_stride;
        to[u] = reinterpret_cast<char*>((uintptr_t)d & ~(uintptr_t)15) + (i - o * t.units) * 16ll;
        const long long before = d - to[u], behind = d + t.bytes - to[u];             // where the row starts and ends, from the word
        first[u] = before > 0 ? (int)before : 0;
        last[u] = i < t.total && behind > first[u] ? (behind < 16 ? (int)behind : 16) : 0;
        shift[u] = 0;
        if (last[u] > first[u]) {
            const char* from = row + (long long)src * t.row_stride - before;        // what belongs at to[u]
            shift[u] = (int)((uintptr_t)from & 15);
            const char* word = from - shift[u];
            if (first[u] + shift[u] < 16) lo[u] = *reinterpret_cast<const uint4*>(word);
            if (last[u] + shift[u] > 16) hi[u] = *reinterpret_cast<const uint4*>(word + 16);
        }
    }
#pragma unroll
    for (int u = 0; u < SHIFT_LOADS; ++u) {
        if (last[u] <= first[u]) continue;
        unsigned w[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
        if (shift[u] & 8) {
#pragma unroll
            for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
        }
        if (shift[u] & 4) {
#pragma unroll
            for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
        }
        uint4 v;
        const int bits = (shift[u] & 3) * 8;
        v.x = __funnelshift_r(w[0], w[1], bits);
        v.y = __funnelshift_r(w[1], w[2], bits);
        v.z = __funnelshift_r(w[2], w[3], bits);
        v.w = __funnelshift_r(w[3], w[4], bits);
        if (first[u] == 0 && last[u] == 16) *reinterpret_cast<uint4*>(to[u]) = v;
        else {
            const unsigned q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const unsigned b = q[k / 4] >> (k % 4 * 8);
                if (t.unit == 1) {
                    if (k >= first[u] && k < last[u]) to[u][k] = (char)b;
                    if (k + 1 >= first[u] && k + 1 < last[u]) to[u][k + 1] = (char)(b >> 8);
                } else if (k >= first[u] && k < last[u]) {
                    *reinterpret_cast<unsigned short*>(to[u] + k) = (unsigned short)b;
                }
            }
        }
    }
}

// Grid (blocks of a row over all tensors, pairs): row dst[y] becomes row src[y].  A pair with a negative index, or of a row with itself, is passed over.
// Bound by memory: 1,000 pages of 0.9 MB take 280 us (6.5 TB/s, as a plain copy), 128 of 0.46 MB 21 (18 at that rate, and a launch).  16 KB a block, four loads a thread
// under way, eight blocks to a multiprocessor.
// SHIFTED: sizes, strides and starts that are no multiples of 16 bytes.  1,201 rows of 9 x 1,358 bytes in pairs of bytes take 16.1 us, so 9.2.
template <bool SHIFTED>
__global__ void __launch_bounds__(ROWS_THREADS) copy_rows_kernel(RowTensors ts, const int* __restrict__ src, const int* __restrict__ dst) {
    pdl_launch_dependents();
    const RowTensor t = ts.t[rows_tensor(ts, blockIdx.x)];
    pdl_wait();
    const int s = src[blockIdx.y], d = dst[blockIdx.y];
    if (s < 0 || d < 0 || s == d) return;
    if (s >= t.rows || d >= t.rows) {
        // (one block of the tensor counts)
        if (threadIdx.x == 0 && blockIdx.x == t.first) atomicAdd(&g_rows_missed, 1u);
        return;
    }
    if (SHIFTED) copy_shifted(t, blockIdx.x - t.first, s, d);
    else copy_aligned(t, blockIdx.x - t.first, s, d);
}

// What a group's blocks have to do, in order: row to[i] becomes row from[i].  from -1: the row that was put aside; to -1: puts the row aside.
struct RowMoves {
    int n;
    int from[2 * ROWS_BEAMS], to[2 * ROWS_BEAMS];
};

// Piece `piece` of a row in one outer entry: ROWS_SPAN units, or what is left of the row.  aside: a place in shared memory for every unit.
template <typename U>
__device__ __forceinline__ void move_units(const RowTensor& t, int piece, const RowMoves& m, uint4* aside) {
    const int pieces = (t.units + ROWS_SPAN - 1) / ROWS_SPAN, o = piece / pieces;
    const unsigned i0 = (unsigned)(piece - o * pieces) * ROWS_SPAN + threadIdx.x;
    U* base = reinterpret_cast<U*>(t.base + (long long)o * t.outer_stride) + i0;
    const int left = (int)(t.units - i0);
    const long long step = t.row_stride / (long long)sizeof(U);
    for (int k = 0; k < m.n; ++k) {
        const int from = m.from[k], to = m.to[k];
        const U* src = from < 0 ? reinterpret_cast<const U*>(aside) + threadIdx.x : base + from * step;
        U* dst = to < 0 ? reinterpret_cast<U*>(aside) + threadIdx.x : base + to * step;
        U v[ROWS_LOADS];
#pragma unroll
        for (int u = 0; u < ROWS_LOADS; ++u)
            if (u * ROWS_THREADS < left) v[u] = src[u * ROWS_THREADS];
#pragma unroll
        for (int u = 0; u < ROWS_LOADS; ++u)
            if (u * ROWS_THREADS < left) dst[u * ROWS_THREADS] = v[u];
    }
}

// Grid (pieces of a row over all tensors, groups): rows slots[g, p] become what rows slots[g, parents[g, p]] were, at once.  A block works out the order of
// its group's moves and makes them in its piece of the rows: every byte is read and written by one thread, and a row is overwritten after all that
// read it have; one row of a cycle is put aside.
// One short piece a block: what is read and written at one time lies close together.  32 of 64 states of 26 MB: 254 us (6.6 TB/s, as a plain copy); blocks that stay and go over many pieces take 284, two moves' loads at a time in fewer blocks 290, all moves' loads at once in two blocks 327.
// Rows that are no multiples of 16 bytes go in units of 8, 4, 2 or 1, a load each: 32 of 64 rows of 1 MB in 24 entries and 0, 8, 4, 2, 1 bytes more take 243, 257, 342,
// 580, 1,074 us (246 at the rate of a plain copy).  The states of all architectures here are float32: 4 bytes at least.
__global__ void __launch_bounds__(ROWS_THREADS) reorder_rows_kernel(RowTensors ts, const int* __restrict__ slots, const int* __restrict__ parents, int places) {
    pdl_launch_dependents();
    __shared__ RowMoves moves;
    __shared__ unsigned readers[ROWS_BEAMS];
    __shared__ uint4 aside[ROWS_SPAN];
    const RowTensor t = ts.t[rows_tensor(ts, blockIdx.x)];
    pdl_wait();
    if (threadIdx.x < 32) {
        const int p = threadIdx.x;
        const int slot = p < places ? slots[blockIdx.y * places + p] : -1, parent = p < places ? parents[blockIdx.y * places + p] : p;
        int from = __shfl_sync(0xffffffffu, slot, parent & 31);
        bool wanted = p < places && parent != p;
        if (wanted && (parent < 0 || parent >= places || slot < 0 || slot >= ts.rows || from < 0 || from >= ts.rows)) {
            if (blockIdx.x == 0) atomicAdd(&g_rows_missed, 1u);          // (one block of the group counts)
            wanted = false;
        }
        // the places that wait to take over what place p holds
        readers[p] = 0u;
        __syncwarp();
        const unsigned same = __match_any_sync(0xffffffffu, wanted ? parent : 32 + p);
        if (wanted) readers[parent] = same;
        __syncwarp();
        unsigned waiting = readers[p];
        unsigned todo = __ballot_sync(0xffffffffu, wanted);
        int n = 0;
        while (todo) {
            const unsigned ready = __ballot_sync(0xffffffffu, ((todo >> p) & 1u) && !(waiting & todo));
            if (ready) {
                if ((ready >> p) & 1u) {
                    const int at = n + __popc(ready & ((1u << p) - 1u));
                    moves.from[at] = from;
                    moves.to[at] = slot;
                }
                n += __popc(ready);
                todo &= ~ready;
            } else {
                // cycles are left, in which every place is read once: what the first holds is put aside for its reader, which is done before
                // another row is put aside
                const int aside = __ffs(todo) - 1;
                if (p == aside) {
                    moves.from[n] = slot;
                    moves.to[n] = -1;
                    waiting = 0u;
                }
                if (((todo >> p) & 1u) && parent == aside) from = -1;
                ++n;
            }
        }
        if (p == 0) moves.n = n;
    }
    __syncthreads();
    if (moves.n == 0) return;
    const int piece = blockIdx.x - t.first;
    if (t.unit == 16) move_units<uint4>(t, piece, moves, aside);
    else if (t.unit == 8) move_units<uint2>(t, piece, moves, aside);
    else if (t.unit == 4) move_units<unsigned>(t, piece, moves, aside);
    else if (t.unit == 2) move_units<unsigned short>(t, piece, moves, aside);
    else move_units<unsigned char>(t, piece, moves, aside);
}

// How a launch divides rows: in blocks of 16-byte units over all outer entries (aligned tensors, or the others), or in pieces within an entry.
enum RowWork { ROWS_ALIGNED, ROWS_SHIFTED, ROWS_PIECES };

// What a launch needs to know of n tensors.  of: six numbers for each - address, outer entries, rows, bytes between outer entries, bytes between rows, bytes
// of a row.  Tensors that are not for this kind of work are left out.  Returns the blocks (x) of the launch, or a negative code.
static long long rows_describe(const long long* of, int n, RowTensors& ts, RowWork work) {
    ts.n = 0;
    ts.rows = 0x7fffffff;
    long long blocks = 0;
    for (int i = 0; i < n; ++i) {
        const long long base = of[6 * i], outer = of[6 * i + 1], rows = of[6 * i + 2], outer_stride = of[6 * i + 3], row_stride = of[6 * i + 4], bytes = of[6 * i + 5];
        if (outer < 1 || rows < 1 || bytes < 1) continue;
        if (rows > 0x7fffffffll || outer_stride < 0 || row_stride < 0) return PICO_ERR_SIZE;
        const long long all = base | bytes | (outer > 1 ? outer_stride : 0) | (rows > 1 ? row_stride : 0);
        const int unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
        if (work != ROWS_PIECES && (unit == 16) != (work == ROWS_ALIGNED)) continue;
        const long long units = work == ROWS_SHIFTED ? (bytes + 30) / 16 : bytes / unit;
        if (units > 0x7fffffffll / outer) return PICO_ERR_SIZE;
        RowTensor& t = ts.t[ts.n++];
        t.base = reinterpret_cast<char*>(base);
        t.outer_stride = outer_stride;
        t.row_stride = row_stride;
        t.bytes = bytes;
        t.units = (unsigned)units;
        t.total = t.units * (unsigned)outer;
        t.rows = (int)rows;
        if (t.rows < ts.rows) ts.rows = t.rows;
        t.unit = unit;
        t.first = (int)blocks;
        const int span = work == ROWS_SHIFTED ? SHIFT_SPAN : ROWS_SPAN;
        blocks += work == ROWS_PIECES ? outer * ((units + span - 1) / span) : (t.total + span - 1ll) / span;
        if (blocks > 0x7fffffffll) return PICO_ERR_SIZE;
    }
    return blocks;
}

PICO_API int pico_copy_rows(const long long* of, int n, const int* src, const int* dst, int pairs, cudaStream_t stream) {
    if (n > ROWS_TENSORS || pairs < 0) return PICO_ERR_SIZE;
    RowTensors aligned, shifted;
    const long long a = rows_describe(of, n, aligned, ROWS_ALIGNED), b = rows_describe(of, n, shifted, ROWS_SHIFTED);
    if (a < 0 || b < 0) return PICO_ERR_SIZE;
    for (int p0 = 0; p0 < pairs; p0 += 65535) {
        const int m = pairs - p0 < 65535 ? pairs - p0 : 65535;
        if (a) pico_launch(copy_rows_kernel<false>, dim3((unsigned)a, m), dim3(ROWS_THREADS), 0, stream, aligned, src + p0, dst + p0);
        if (b) pico_launch(copy_rows_kernel<true>, dim3((unsigned)b, m), dim3(ROWS_THREADS), 0, stream, shifted, src + p0, dst + p0);
    }
    return pico_launch_status();
}

PICO_API int pico_reorder_rows(const long long* of, int n, const int* slots, const int* parents, int groups, int places, cudaStream_t stream) {
    if (n > ROWS_TENSORS || groups < 0 || places < 1 || places > ROWS_BEAMS) return PICO_ERR_SIZE;
    RowTensors ts;
    const long long blocks = rows_describe(of, n, ts, ROWS_PIECES);
    if (blocks < 0) return (int)blocks;
    if (blocks == 0) return 0;
    for (int g0 = 0; g0 < groups; g0 += 65535) {
        const int m = groups - g0 < 65535 ? groups - g0 : 65535;
        pico_launch(reorder_rows_kernel, dim3((unsigned)blocks, m), dim3(ROWS_THREADS), 0, stream, ts, slots + (long long)g0 * places,
                    parents + (long long)g0 * places, places);
    }
    return pico_launch_status();
}
