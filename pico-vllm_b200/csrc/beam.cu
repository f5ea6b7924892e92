// The choice of beam search: which beams of a request go on, and with which token.
//
// With x[b, t] the logits of the request's beams and s[b] their scores (sums of log-probabilities), a candidate (b, t) is worth
//     v[b, t] = s[b] + x[b, t] - log sum_u exp x[b, u].
// Candidates whose v is a finite number are ranked by (v descending, b * V + t ascending).  A row that holds no number or an infinity, or is
// masked whole, has a normaliser that is none, and none of its tokens is a candidate; nor is one of a beam whose score is -infinity.
// Going down the ranks, a candidate with the end token sets its beam's hypothesis aside if it is among the B best; the first B of the others
// go on.  Of these the best child of beam p takes place p (its cache stays where it is), the others in their order the places that are left.
#include "common.cuh"

#define BEAM_THREADS 256
#define BEAM_LOADS 4                                            // 16-byte loads of a thread under way
#define BEAM_TILE (BEAM_THREADS * 4 * BEAM_LOADS)               // elements that a block takes at a time
#define BEAM_MAX 32                                             // beams of a request: lanes of the warp that ranks
#define BEAM_LIST (2 * BEAM_MAX + BEAM_TILE / 4 + 64)           // candidates that wait in shared memory (see beam_rows_kernel)

typedef unsigned long long u64;

// A logit and its place as one whole number that is ordered as (logit, earlier place); 0 is below all of them.  -0 counts as 0.
__device__ __forceinline__ u64 beam_key(float x, unsigned at) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return ((u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xffffffffu - at);
}
__device__ __forceinline__ float beam_key_logit(u64 key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int beam_key_at(u64 key) { return (int)(0xffffffffu - (unsigned)key); }

// Grid (parts, rows).  Block (p, r) reads elements [p * per, (p + 1) * per) of row r once (per: a multiple of the tile) and leaves their
// largest, the sum of exp(x - largest) and their K best, in order.
// VEC: rows start on 16 bytes; without it the same elements go to the same threads, so that rows of equal numbers have equal sums wherever
// they lie.
template <bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS, 4)
beam_rows_kernel(const float* __restrict__ logits, long long row_stride, int V, int K, int groups, int per, u64* __restrict__ best,
                 float2* __restrict__ sums) {
    pdl_launch_dependents();
    __shared__ u64 list[BEAM_LIST];
    __shared__ u64 sorted[2 * BEAM_MAX];
    __shared__ u64 tops[BEAM_THREADS];
    __shared__ float scratch[33];
    __shared__ int s_n;
    __shared__ float s_limit;
    __shared__ u64 s_raise;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const int p0 = min(V, part * per), p1 = min(V, p0 + per);
    const float* x = logits + (long long)r * row_stride;
    if (tid == 0) { s_n = 0; s_limit = -INFINITY; }
    __syncthreads();
    pdl_wait();
    constexpr float LOG2E = 1.4426950408889634f;
    float m = -INFINITY, s = 0.f, limit = -INFINITY;
    float next[4 * BEAM_LOADS];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int u = 0; u < BEAM_LOADS; ++u) {
            const int i = t0 + (u * BEAM_THREADS + tid) * 4;
            if (VEC && i + 3 < p1) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(x + i));
                next[4 * u] = q.x; next[4 * u + 1] = q.y; next[4 * u + 2] = q.z; next[4 * u + 3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) next[4 * u + e] = i + e < p1 ? __ldg(x + i + e) : -INFINITY;
            }
        }
    };
    if (p0 < p1) fetch(p0);
    for (int t0 = p0; t0 < p1; t0 += BEAM_TILE) {
        float v[4 * BEAM_LOADS];
#pragma unroll
        for (int i = 0; i < 4 * BEAM_LOADS; ++i) v[i] = next[i];
        if (t0 + BEAM_TILE < p1) fetch(t0 + BEAM_TILE);
        float tmax = v[0];
#pragma unroll
        for (int i = 1; i < 4 * BEAM_LOADS; ++i) tmax = fmaxf(tmax, v[i]);
        if (tmax > m) {
            s *= exp2f((m - tmax) * LOG2E);
            m = tmax;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float add = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * BEAM_LOADS; ++i) add += exp2f((v[i] - ref) * LOG2E);
        s += add;
        // ---- candidates: what is above the K-th best so far (later elements lose to equal earlier ones)
        const int above = __syncthreads_count(tmax > limit);
        if (above == 0) continue;
        u64 raise = 0ull;
        if (above > K) {
            // many: the K-th largest of `groups` >= 4 K maxima, each of as many threads, bounds the K-th best from below, and at most
            // (K - 1) * TILE / groups + 1 elements reach it
            u64 top = 0ull;
#pragma unroll
            for (int i = 4 * BEAM_LOADS - 1; i >= 0; --i)
                if (v[i] == tmax) top = beam_key(tmax, t0 + ((i >> 2) * BEAM_THREADS + tid) * 4 + (i & 3));
            if (!(tmax > limit)) top = 0ull;
            const int each = BEAM_THREADS / groups;
            for (int o = 1; o < each; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (tid % each == 0) tops[tid / each] = top;
            if (tid == 0) s_raise = 0ull;
            __syncthreads();
            if (tid < groups) {
                const u64 mine = tops[tid];
                int rank = 0;
                for (int j = 0; j < groups; ++j) rank += tops[j] > mine;
                if (rank == K - 1 && mine) s_raise = mine;
            }
            __syncthreads();
            raise = s_raise;
        }
        if (tmax > limit) {
#pragma unroll
            for (int i = 0; i < 4 * BEAM_LOADS; ++i)
                if (v[i] > limit) {
                    const u64 key = beam_key(v[i], t0 + ((i >> 2) * BEAM_THREADS + tid) * 4 + (i & 3));
                    if (key >= raise) list[atomicAdd(&s_n, 1)] = key;
                }
        }
        __syncthreads();
        const int n = s_n;
        if (n > K) {                        // the K best of them, in order
            for (int i = tid; i < n; i += BEAM_THREADS) {
                const u64 mine = list[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += list[j] > mine;
                if (rank < K) sorted[rank] = mine;
            }
            __syncthreads();
            if (tid < K) list[tid] = sorted[tid];
            if (tid == 0) { s_n = K; s_limit = beam_key_logit(sorted[K - 1]); }
            __syncthreads();
            limit = s_limit;
        }
    }
    // ---- the part's results
    const int n = s_n;
    if (tid < K) sorted[tid] = 0ull;
    const float top = block_max(m, scratch);
    const float sum = block_sum(m == -INFINITY ? s : s * exp2f((m - top) * LOG2E), scratch);
    for (int i = tid; i < n; i += BEAM_THREADS) {
        const u64 mine = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > mine;
        if (rank < K) sorted[rank] = mine;
    }
    __syncthreads();
    const size_t at = (size_t)r * gridDim.x + part;
    if (tid < K) best[at * K + tid] = sorted[tid];
    if (tid == 0) sums[at] = make_float2(top, sum);
}

// The largest of a warp's 64-bit numbers, in every lane.
__device__ __forceinline__ u64 beam_warp_max(u64 v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return ((u64)hi << 32) | lo;
}

// Grid (groups), a warp for each of the group's rows.  Warp b merges the lists of row b's parts, then the first warp ranks the rows' lists
// against one another, a lane for each row, until B candidates that go on are found.
__global__ void beam_join_kernel(const u64* __restrict__ best, const float2* __restrict__ sums, int parts, int K, int V, int rows, int beams,
                                 int end_token, const float* scores, int* tokens, int* parents, float* out_scores, float* ended) {
    pdl_launch_dependents();
    __shared__ u64 lists[BEAM_MAX][2 * BEAM_MAX];
    __shared__ double offsets[BEAM_MAX], tops[BEAM_MAX];
    extern __shared__ __align__(16) unsigned char beam_smem[];
    u64* keys = reinterpret_cast<u64*>(beam_smem);                                       // [rows][parts][K]
    unsigned char* heads = beam_smem + (size_t)rows * parts * K * sizeof(u64);           // [rows][parts]: how many of a list are taken
    const int g = blockIdx.x, lane = threadIdx.x & 31, b = threadIdx.x >> 5;
    pdl_wait();
    {
        const size_t first = ((size_t)g * rows + b) * parts;
        u64* mine = keys + (size_t)b * parts * K;
        unsigned char* taken = heads + b * parts;
        for (int i = lane; i < parts * K; i += 32) mine[i] = best[first * K + i];
        float top = -INFINITY;
        for (int p = lane; p < parts; p += 32) {
            taken[p] = 0;
            top = fmaxf(top, sums[first + p].x);
        }
        top = warp_max(top);
        double sum = 0.0;
        for (int p = lane; p < parts; p += 32) {
            const float2 q = sums[first + p];
            sum += q.x == -INFINITY ? (double)q.y : (double)q.y * (double)expf(q.x - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        // v = (x - largest) + (s - log sum): as near to s as it gets, however large the logits are
        const double off = (double)scores[g * rows + b] - log(sum);
        if (lane == 0) { offsets[b] = off; tops[b] = (double)top; }
        __syncwarp();
        u64* out = lists[b];
        if (!isfinite(off)) {
            for (int k = lane; k < K; k += 32) out[k] = 0ull;
        } else if (parts == 1) {
            for (int k = lane; k < K; k += 32) out[k] = mine[k];
        } else {
            // a lane has the lists of parts lane, lane + 32, ..; their largest head against the other lanes', K times
            u64 head = 0ull;
            int from = 0;
            auto look = [&]() {
                head = 0ull;
                for (int p = lane; p < parts; p += 32) {
                    const u64 c = taken[p] < K ? mine[p * K + taken[p]] : 0ull;
                    if (c > head) { head = c; from = p; }
                }
            };
            look();
            for (int k = 0; k < K; ++k) {
                const u64 w = beam_warp_max(head);
                if (lane == 0) out[k] = w;
                if (w != 0ull && head == w) {
                    ++taken[from];
                    look();
                }
            }
        }
    }
    __syncthreads();
    if (b != 0) return;
    const unsigned all = beams == 32 ? 0xffffffffu : (1u << beams) - 1u;
    const double off = lane < rows ? offsets[lane] : 0.0, row_top = lane < rows ? tops[lane] : 0.0;
    int k = 0;
    u64 value = 0ull;                   // of the row's best candidate that is left, as a whole number that is ordered as it
    double v = 0.0;
    int token = 0;
    auto head = [&]() {
        const u64 key = lane < rows && k < K ? lists[lane][k] : 0ull;
        value = 0ull;
        if (key == 0ull) return;
        v = ((double)beam_key_logit(key) - row_top) + off;
        token = beam_key_at(key);
        const u64 bits = (u64)__double_as_longlong(v + 0.0);
        value = bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
    };
    head();
    double end_value = -INFINITY, my_value = -INFINITY;
    int my_token = -1, my_parent = -1, count = 0;
    unsigned has = 0u;                  // parents with a child
    bool extra = lane < beams;
    for (int rank = 0; count < beams && rank < 2 * beams; ++rank) {
        const u64 w = beam_warp_max(value);
        if (w == 0ull) break;
        const int who = __ffs(__ballot_sync(0xffffffffu, value == w)) - 1;        // of equal ones the first beam
        const int t = __shfl_sync(0xffffffffu, token, who);
        const double d = __shfl_sync(0xffffffffu, v, who);
        if (t == end_token) {
            if (lane == who && rank < beams) end_value = d;
        } else {
            if (lane == count) {
                my_value = d; my_token = t; my_parent = who;
                extra = (has >> who) & 1u;
            }
            has |= 1u << who;
            ++count;
        }
        if (lane == who) { ++k; head(); }
    }
    // places: the first child of a parent has the parent's, the others (and those that hold nothing) the ones that are left
    const unsigned others = __ballot_sync(0xffffffffu, extra);
    if (lane < beams) {
        int place = my_parent;
        if (extra) {
            unsigned left = all & ~has;
            for (int e = __popc(others & ((1u << lane) - 1u)); e > 0; --e) left &= left - 1u;
            place = __ffs(left) - 1;
        }
        const int at = g * beams + place;
        tokens[at] = my_token;
        parents[at] = my_token < 0 ? place : my_parent;
        out_scores[at] = (float)my_value;
    }
    if (lane < rows) ended[g * rows + lane] = (float)end_value;
}

#define BEAM_JOIN_KEYS 20480    // candidates that a block of beam_join_kernel has room for in shared memory (160 KB)

// Parts of a row: as many as run at once over all rows, none shorter than a tile, and no more than the join has room for.
static int beam_parts(int groups, int rows, int V, int K) {
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE;
    int want = (4 * pico_num_sms()) / (groups * rows);
    if (want > BEAM_JOIN_KEYS / (rows * K)) want = BEAM_JOIN_KEYS / (rows * K);
    const int parts = want < 1 ? 1 : want > tiles ? tiles : want;
    const int each = (tiles + parts - 1) / parts;
    return (tiles + each - 1) / each;
}
static int beam_candidates(int beams, int end_token) { return end_token >= 0 ? 2 * beams : beams; }
static bool beam_takes(int groups, int rows, int V, int beams) {
    return groups >= 1 && rows >= 1 && rows <= beams && beams <= BEAM_MAX && V >= 1 && (long long)groups * rows <= 65535 &&
           (long long)rows * V <= 0x7fffffffll;
}

// Bytes of scratch that pico_beam_select needs (its start on 16 bytes); negative: a size it does not take.
PICO_API long long pico_beam_scratch(int groups, int rows, int V, int beams, int end_token) {
    if (!beam_takes(groups, rows, V, beams)) return PICO_ERR_SIZE;
    const int K = beam_candidates(beams, end_token);
    return (long long)groups * rows * beam_parts(groups, rows, V, K) * (8ll * K + 8);
}

// logits: [groups * rows, row_stride] float32, the first V columns are used; scores: [groups, rows].  tokens, parents, out_scores: [groups, beams];
// ended: [groups, rows].  end_token < 0: none.  out_scores may be scores where rows == beams.
PICO_API int pico_beam_select(const float* logits, long long row_stride, int groups, int rows, int V, int beams, int end_token, const float* scores,
                              void* scratch, int* tokens, int* parents, float* out_scores, float* ended, cudaStream_t stream) {
    if (!beam_takes(groups, rows, V, beams)) return PICO_ERR_SIZE;
    const int K = beam_candidates(beams, end_token), R = groups * rows, parts = beam_parts(groups, rows, V, K);
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE, per = (tiles + parts - 1) / parts * BEAM_TILE;
    int sets = 32;
    while (sets < 4 * K && sets < BEAM_THREADS) sets *= 2;
    u64* best = reinterpret_cast<u64*>(scratch);
    float2* sums = reinterpret_cast<float2*>(best + (size_t)R * parts * K);
    const bool vec = row_stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    const size_t smem = (size_t)rows * parts * (K * sizeof(u64) + 1);
    if (smem > 24 * 1024) {             // beside the kernel's own 17 KB
        const cudaError_t e = cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)cudaGetLastError();
    }
    if (vec) pico_launch(beam_rows_kernel<true>, dim3(parts, R), dim3(BEAM_THREADS), 0, stream, logits, row_stride, V, K, sets, per, best, sums);
    else pico_launch(beam_rows_kernel<false>, dim3(parts, R), dim3(BEAM_THREADS), 0, stream, logits, row_stride, V, K, sets, per, best, sums);
    const int status = pico_launch_status();
    if (status) return status;
    pico_launch(beam_join_kernel, dim3(groups), dim3(32 * rows), smem, stream, (const u64*)best, (const float2*)sums, parts, K, V, rows, beams, end_token,
                scores, tokens, parents, out_scores, ended);
    return pico_launch_status();
}
