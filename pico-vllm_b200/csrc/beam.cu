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

// 2^x; results below 2^-126 are 0
__device__ __forceinline__ float beam_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Grid (parts, rows).  Block (p, r) reads elements [p * per, (p + 1) * per) of row r once (per: a multiple of the tile) and leaves their
// largest, the sum of exp(x - largest) and their K best, in order.
// Each thread keeps a running maximum and sum of its own elements.  Candidates wait unsorted in shared memory: an element joins them if it is above
// `limit`, a lower bound of the K-th best so far.  Of the first tile the bound comes from maxima of groups of threads; later tiles bring a few
// candidates each (K / j the j-th of random ones), and only when some have gathered are the K best picked out and the bound raised.
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
    __shared__ float2 warp_sums[BEAM_THREADS / 32];
    __shared__ int s_n;
    __shared__ u64 s_raise;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const int p0 = min(V, part * per), p1 = min(V, p0 + per);
    const float* x = logits + (long long)r * row_stride;
    if (tid == 0) s_n = 0;
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
    // the K best of the n candidates into `sorted`, in order (what is above the n-th is left as it was)
    auto rank = [&](int n) {
        for (int i = tid; i < n; i += BEAM_THREADS) {
            const u64 mine = list[i];
            int better = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) better += list[j] > mine;
            if (better < K) sorted[better] = mine;
        }
        __syncthreads();
    };
    int gathered = 0, room = BEAM_LIST;     // candidates since the last ranking, about; places of the list that are free, at least
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
            s *= beam_exp2((m - tmax) * LOG2E);
            m = tmax;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float add = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * BEAM_LOADS; ++i) add += beam_exp2((v[i] - ref) * LOG2E);
        s += add;
        // ---- candidates (later elements lose to equal earlier ones: what is not above the bound is none)
        const int above = __syncthreads_count(tmax > limit);
        if (above == 0) continue;
        u64 raise = 0ull;
        int most = 4 * BEAM_LOADS * above;
        if (above > K) {
            // many: the K-th largest of `groups` >= 4 K maxima, each of as many threads, bounds the K-th best from below, and at most
            // (K - 1) * TILE / groups + 1 <= TILE / 4 elements reach it
            u64 top = 0ull;
            if (tmax > limit) {
#pragma unroll
                for (int i = 4 * BEAM_LOADS - 1; i >= 0; --i)
                    if (v[i] == tmax) top = beam_key(tmax, t0 + ((i >> 2) * BEAM_THREADS + tid) * 4 + (i & 3));
            }
            const int each = BEAM_THREADS / groups;
            for (int o = 1; o < each; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (tid % each == 0) tops[tid / each] = top;
            if (tid == 0) s_raise = 0ull;
            __syncthreads();
            if (tid < groups) {
                const u64 mine = tops[tid];
                int better = 0;
#pragma unroll 8
                for (int j = 0; j < groups; ++j) better += tops[j] > mine;
                if (better == K - 1 && mine) s_raise = mine;
            }
            __syncthreads();
            raise = s_raise;
            most = BEAM_TILE / 4;
        }
        if (most > room) {                  // pick out the K best first
            const int n = s_n;
            rank(n);
            if (tid < min(n, K)) list[tid] = sorted[tid];
            if (tid == 0) s_n = min(n, K);
            if (n >= K) limit = fmaxf(limit, beam_key_logit(sorted[K - 1]));
            gathered = 0;
            room = BEAM_LIST - K;
            __syncthreads();
        }
        if (tmax > limit) {
#pragma unroll
            for (int i = 0; i < 4 * BEAM_LOADS; ++i)
                if (v[i] > limit) {
                    const u64 key = beam_key(v[i], t0 + ((i >> 2) * BEAM_THREADS + tid) * 4 + (i & 3));
                    if (key >= raise) list[atomicAdd(&s_n, 1)] = key;
                }
        }
        room -= most;
        gathered += min(above, 2 * K);
        if (raise) limit = beam_key_logit(raise);
        if (gathered > 3 * K) {
            __syncthreads();
            const int n = s_n;
            if (n > K) {
                rank(n);
                limit = fmaxf(limit, beam_key_logit(sorted[K - 1]));
                if (tid < K) list[tid] = sorted[tid];
                if (tid == 0) s_n = K;
            }
            gathered = 0;
            room = BEAM_LIST - min(n, K);
            // (the barrier before the next candidates is the next tile's)
        }
    }
    // ---- the part's results
    float top = warp_max(m);
    float sum = warp_sum(m == -INFINITY ? s : s * beam_exp2((m - top) * LOG2E));
    if ((tid & 31) == 0) warp_sums[tid >> 5] = make_float2(top, sum);
    __syncthreads();
    const int n = s_n;
    if (tid < K) sorted[tid] = 0ull;
    __syncthreads();
    rank(n);
    const size_t at = (size_t)r * gridDim.x + part;
    if (tid < K) best[at * K + tid] = sorted[tid];
    if (tid < 32) {
        const float2 q = tid < BEAM_THREADS / 32 ? warp_sums[tid] : make_float2(-INFINITY, 0.f);
        top = warp_max(q.x);
        sum = warp_sum(q.x == -INFINITY ? q.y : q.y * beam_exp2((q.x - top) * LOG2E));
        if (tid == 0) sums[at] = make_float2(top, sum);
    }
}

// The largest of a warp's 64-bit numbers, in every lane.
__device__ __forceinline__ u64 beam_warp_max(u64 v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return ((u64)hi << 32) | lo;
}

// A finite number as a whole one that is ordered as it and above 0 (-0 counts as 0), and back.
__device__ __forceinline__ u64 beam_order(double v) {
    const u64 bits = (u64)__double_as_longlong(v + 0.0);
    return bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}
__device__ __forceinline__ double beam_unorder(u64 o) { return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o)); }

// Grid (groups), a warp for each of the group's rows (four at least: all of them fetch).  Warp b merges the lists of row b's parts, a lane for every
// 32nd of them, then the first warp ranks the rows' lists against one another, a lane for each row, until B candidates that go on are found: what a
// round waits for are the two warp-wide maxima and the winner's next number, which is there already.
__global__ void beam_join_kernel(const u64* __restrict__ best, const float2* __restrict__ sums, int parts, int K, int rows, int beams, int end_token,
                                 const float* scores, int* tokens, int* parents, float* out_scores, float* ended) {
    pdl_launch_dependents();
    __shared__ u64 values[BEAM_MAX][2 * BEAM_MAX];              // of the rows' best, in order
    __shared__ int places[BEAM_MAX][2 * BEAM_MAX];              // their tokens
    __shared__ int ends[BEAM_MAX];                              // which of them is the end token
    extern __shared__ __align__(16) unsigned char beam_smem[];
    u64* keys = reinterpret_cast<u64*>(beam_smem);                                       // [rows][parts][K]
    unsigned char* heads = beam_smem + (size_t)rows * parts * K * sizeof(u64);           // [rows][parts]: how many of a list are taken
    const int g = blockIdx.x, lane = threadIdx.x & 31, b = threadIdx.x >> 5;
    pdl_wait();
    {
        const u64* from = best + (size_t)g * rows * parts * K;
        const unsigned to = (unsigned)__cvta_generic_to_shared(keys);
#pragma unroll 8
        for (int i = threadIdx.x; i < rows * parts * K; i += blockDim.x)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to + 8u * i), "l"(from + i) : "memory");
    }
    double off = 0.0, row_top = 0.0;
    if (b < rows) {
        // v = (x - largest) + (s - log sum): as near to s as it gets, however large the logits are
        const float2* q = sums + ((size_t)g * rows + b) * parts;
        const float score = scores[g * rows + b];
        float top = -INFINITY;
        double sum = 0.0;
#pragma unroll 2
        for (int p = lane; p < parts; p += 32) {
            const float2 c = q[p];
            if (c.x > top) {
                sum *= (double)expf(top - c.x);
                top = c.x;
            }
            sum += c.x == -INFINITY ? (double)c.y : (double)c.y * (double)expf(c.x - top);
        }
        const float all = warp_max(top);
        if (top != -INFINITY) sum *= (double)expf(top - all);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        off = (double)score - log(sum);
        row_top = (double)all;
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    __syncthreads();
    if (b < rows) {
        u64* mine = keys + (size_t)b * parts * K;
        u64* out = values[b];
        if (!isfinite(off)) {
            for (int k = lane; k < K; k += 32) out[k] = 0ull;
        } else if (parts == 1) {
            for (int k = lane; k < K; k += 32) out[k] = mine[k];
        } else if (parts <= 64) {
            const u64 *q0 = mine + lane * K, *q1 = q0 + 32 * K;
            const bool has0 = lane < parts, has1 = lane + 32 < parts;
            int k0 = 0, k1 = 0;
            u64 c0 = has0 ? q0[0] : 0ull, c1 = has1 ? q1[0] : 0ull, d0 = has0 && K > 1 ? q0[1] : 0ull, d1 = has1 && K > 1 ? q1[1] : 0ull;
            for (int k = 0; k < K; ++k) {
                const u64 w = beam_warp_max(max(c0, c1));
                if (lane == 0) out[k] = w;
                if (w == 0ull) continue;
                if (c0 == w) {
                    c0 = d0;
                    ++k0;
                    d0 = k0 + 1 < K ? q0[k0 + 1] : 0ull;
                } else if (c1 == w) {
                    c1 = d1;
                    ++k1;
                    d1 = k1 + 1 < K ? q1[k1 + 1] : 0ull;
                }
            }
        } else {
            unsigned char* taken = heads + b * parts;
            for (int p = lane; p < parts; p += 32) taken[p] = 0;
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
        __syncwarp();
        if (lane == 0) ends[b] = -1;
        __syncwarp();
        for (int k = lane; k < K; k += 32) {
            const u64 key = out[k];
            const int t = beam_key_at(key);
            out[k] = key ? beam_order(((double)beam_key_logit(key) - row_top) + off) : 0ull;
            places[b][k] = t;
            if (key && t == end_token) ends[b] = k;
        }
    }
    __syncthreads();
    if (b != 0) return;
    const u64* list = values[lane < rows ? lane : 0];
    const int end_at = lane < rows ? ends[lane] : -1;
    int k = 0;
    u64 value = lane < rows ? list[0] : 0ull, next = lane < rows && K > 1 ? list[1] : 0ull;
    int my_parent = -1, my_k = 0, end_k = -1, count = 0;
    unsigned has = 0u;                  // parents with a child
    bool extra = lane < beams;
    for (int rank = 0; count < beams && rank < K; ++rank) {
        const u64 w = beam_warp_max(value);
        if (w == 0ull) break;
        const int who = __ffs(__ballot_sync(0xffffffffu, value == w)) - 1;        // of equal ones the first beam
        const bool won = lane == who;
        const int at = __shfl_sync(0xffffffffu, k, who);
        if (__any_sync(0xffffffffu, won && k == end_at)) {
            if (won && rank < beams) end_k = k;
        } else {
            if (lane == count) {
                my_parent = who;
                my_k = at;
                extra = (has >> who) & 1u;
            }
            has |= 1u << who;
            ++count;
        }
        if (won) {
            value = next;
            ++k;
            next = k + 1 < K ? list[k + 1] : 0ull;
        }
    }
    // places: the first child of a parent has the parent's, the others (and those that hold nothing) the ones that are left
    const unsigned others = __ballot_sync(0xffffffffu, extra);
    if (lane < beams) {
        int place = my_parent;
        if (extra) {
            unsigned left = (beams == 32 ? 0xffffffffu : (1u << beams) - 1u) & ~has;
            for (int e = __popc(others & ((1u << lane) - 1u)); e > 0; --e) left &= left - 1u;
            place = __ffs(left) - 1;
        }
        const int at = g * beams + place;
        tokens[at] = my_parent < 0 ? -1 : places[my_parent][my_k];
        parents[at] = my_parent < 0 ? place : my_parent;
        out_scores[at] = my_parent < 0 ? -INFINITY : (float)beam_unorder(values[my_parent][my_k]);
    }
    if (lane < rows) ended[g * rows + lane] = end_k < 0 ? -INFINITY : (float)beam_unorder(list[end_k]);
}

#define BEAM_JOIN_KEYS 20480    // candidates that a block of beam_join_kernel has room for in shared memory (160 KB)

// Parts of a row: as many as run at once over all rows, none shorter than a tile, and no more than the join and the scratch have room for.
static int beam_parts(int groups, int rows, int V, int K, long long lists) {
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE, R = groups * rows;
    long long want = (4 * pico_num_sms()) / R;
    if (want > BEAM_JOIN_KEYS / (rows * K)) want = BEAM_JOIN_KEYS / (rows * K);
    if (want > lists / R) want = lists / R;
    const int parts = want < 1 ? 1 : want > tiles ? tiles : (int)want;
    const int each = (tiles + parts - 1) / parts;
    return (tiles + each - 1) / each;
}

// logits: [groups * rows, row_stride] float32, the first V columns are used; scores: [groups, rows].  tokens, parents, out_scores: [groups, beams];
// ended: [groups, rows].  end_token < 0: none.  out_scores may be scores where rows == beams.
// scratch: `lists` lists of 16 * beams + 8 bytes (8 * beams + 8 without an end token), from a 16-byte boundary on; one for each row at least, and 640 let
// rows be read in as many parts as a device of 160 multiprocessors runs at once.
PICO_API int pico_beam_select(const float* logits, long long row_stride, int groups, int rows, int V, int beams, int end_token, const float* scores,
                              void* scratch, int lists, int* tokens, int* parents, float* out_scores, float* ended, cudaStream_t stream) {
    if (groups < 1 || rows < 1 || rows > beams || beams > BEAM_MAX || V < 1 || (long long)groups * rows > 65535 ||
        (long long)rows * V > 0x7fffffffll || lists < groups * rows)
        return PICO_ERR_SIZE;
    const int K = end_token >= 0 ? 2 * beams : beams, R = groups * rows, parts = beam_parts(groups, rows, V, K, lists);
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE, per = (tiles + parts - 1) / parts * BEAM_TILE;
    int sets = 32;
    while (sets < 4 * K && sets < BEAM_THREADS) sets *= 2;
    u64* best = reinterpret_cast<u64*>(scratch);
    float2* sums = reinterpret_cast<float2*>(best + (size_t)R * parts * K);
    const bool vec = row_stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    const size_t smem = (size_t)rows * parts * (K * sizeof(u64) + 1);
    if (smem > 20 * 1024) {             // beside the kernel's own 25 KB
        const cudaError_t e = cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)cudaGetLastError();
    }
    if (vec) pico_launch(beam_rows_kernel<true>, dim3(parts, R), dim3(BEAM_THREADS), 0, stream, logits, row_stride, V, K, sets, per, best, sums);
    else pico_launch(beam_rows_kernel<false>, dim3(parts, R), dim3(BEAM_THREADS), 0, stream, logits, row_stride, V, K, sets, per, best, sums);
    const int status = pico_launch_status();
    if (status) return status;
    pico_launch(beam_join_kernel, dim3(groups), dim3(32 * (rows < 4 ? 4 : rows)), smem, stream, (const u64*)best, (const float2*)sums, parts, K, rows, beams, end_token,
                scores, tokens, parents, out_scores, ended);
    return pico_launch_status();
}
