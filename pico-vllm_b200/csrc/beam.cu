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
#define BEAM_AGAIN 2                                            // ... and of the second look
#define BEAM_MAX 32                                             // beams of a request: lanes of the warp that ranks
#define BEAM_LIST (4 * BEAM_THREADS + 128)                      // candidates that wait in shared memory (see beam_rows_kernel)

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

// two sums, products at a time
__device__ __forceinline__ u64 beam_pair(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 beam_unpair(u64 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ u64 beam_add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 beam_mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Grid (parts, rows).  Block (p, r) reads elements [p * per, (p + 1) * per) of row r (per: a multiple of the tile) and leaves their largest, the sum of
// exp(x - largest) and their K best, in order.
// One pass over the elements keeps, in every thread, the running maximum and sum and the maximum of each of its four columns (the 16-byte loads at
// one place of all tiles); no thread waits for another.  The K-th largest of `groups` >= 2 K maxima of threads then bounds the K-th best from
// below, and only the columns that reach it, a few more than K of 1,024, are read once more (from L2) for the elements themselves.
// Bound by memory where rows are many: 256 of 151,936 (156 MB) take 28 us without the join, 24 at the rate of a plain copy; what follows the pass, 2 to 3 us in
// blocks that end together, is the rest.  Few rows are cut into parts, for which the same steps, some 5,000 cycles, are most of the time.
// VEC: rows start on 16 bytes; otherwise whole words of 16 bytes are read all the same, two for four elements of a thread that lie across them (the second is the
// neighbour's first, and only words with elements of the row are read).  The same elements go to the same threads either way, so that rows of equal
// numbers have equal sums wherever they lie.  504 rows of 50,512 that start anywhere take 31.5 us, by loads of 4 bytes 33.7.
template <bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS, 6)
beam_rows_kernel(const float* __restrict__ logits, long long row_stride, int V, int K, int groups, int per, u64* __restrict__ best,
                 float2* __restrict__ sums) {
    pdl_launch_dependents();
    __shared__ u64 list[BEAM_LIST];
    __shared__ u64 sorted[2 * BEAM_MAX];
    __shared__ __align__(16) float tops[BEAM_THREADS];
    __shared__ unsigned short columns[BEAM_THREADS * BEAM_LOADS];
    __shared__ float2 warp_sums[BEAM_THREADS / 32];
    __shared__ int s_n, s_columns;
    __shared__ float s_bound;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const int p0 = min(V, part * per), p1 = min(V, p0 + per);
    const float* x = logits + (long long)r * row_stride;
    if (tid == 0) { s_n = 0; s_columns = 0; s_bound = -INFINITY; }
    if (tid < K) sorted[tid] = 0ull;
    pdl_wait();
    constexpr float LOG2E = 1.4426950408889634f;
    float m = -INFINITY, s = 0.f, column[BEAM_LOADS];
#pragma unroll
    for (int u = 0; u < BEAM_LOADS; ++u) column[u] = -INFINITY;
    const int ahead = VEC ? 0 : (int)((uintptr_t)x >> 2) & 3;       // elements of the row's first word of 16 bytes that are not the row's
    auto fetch = [&](float* v, int t0) {
        if (t0 + BEAM_TILE <= p1) {
#pragma unroll
            for (int u = 0; u < BEAM_LOADS; ++u) {
                const float4* q = reinterpret_cast<const float4*>(x - ahead + t0 + (u * BEAM_THREADS + tid) * 4);
                const float4 lo = __ldg(q);
                v[4 * u] = lo.x; v[4 * u + 1] = lo.y; v[4 * u + 2] = lo.z; v[4 * u + 3] = lo.w;
                if (!VEC && ahead) {
                    const float4 hi = __ldg(q + 1);
                    const bool two = ahead & 2, one = ahead & 1;
                    const float a = two ? lo.z : lo.x, b = two ? lo.w : lo.y, c = two ? hi.x : lo.z, d = two ? hi.y : lo.w, f = two ? hi.z : hi.x;
                    v[4 * u] = one ? b : a; v[4 * u + 1] = one ? c : b; v[4 * u + 2] = one ? d : c; v[4 * u + 3] = one ? f : d;
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < BEAM_LOADS; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = t0 + (u * BEAM_THREADS + tid) * 4 + e;
                    v[4 * u + e] = i < p1 ? __ldg(x + i) : -INFINITY;
                }
        }
    };
    auto take = [&](const float* v) {
        float tmax = -INFINITY;
#pragma unroll
        for (int u = 0; u < BEAM_LOADS; ++u) {
            const float q = fmaxf(fmaxf(v[4 * u], v[4 * u + 1]), fmaxf(v[4 * u + 2], v[4 * u + 3]));
            column[u] = fmaxf(column[u], q);
            tmax = fmaxf(tmax, q);
        }
        if (tmax > m) {
            s *= beam_exp2((m - tmax) * LOG2E);
            m = tmax;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const u64 less = beam_pair(-ref, -ref), log2e = beam_pair(LOG2E, LOG2E);
        u64 add = 0ull;
#pragma unroll
        for (int i = 0; i < 4 * BEAM_LOADS; i += 2) {
            const float2 e = beam_unpair(beam_mul2(beam_add2(beam_pair(v[i], v[i + 1]), less), log2e));
            add = beam_add2(add, beam_pair(beam_exp2(e.x), beam_exp2(e.y)));
        }
        const float2 halves = beam_unpair(add);
        s += halves.x + halves.y;
    };
    for (int t0 = p0; t0 < p1; t0 += BEAM_TILE) {
        float v[4 * BEAM_LOADS];
        fetch(v, t0);
        take(v);
    }
    // ---- a bound of the K-th best, and the columns that reach it
    const int each = BEAM_THREADS / groups;
    float top = m;
    for (int o = 1; o < each; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid % each == 0) tops[tid / each] = top;
    top = warp_max(top);
    const float sum = warp_sum(m == -INFINITY ? s : s * beam_exp2((m - top) * LOG2E));
    if ((tid & 31) == 0) warp_sums[tid >> 5] = make_float2(top, sum);
    __syncthreads();
    if (tid < groups) {
        const float mine = tops[tid];
        int larger = 0, equal = 0;
#pragma unroll 4
        for (int j = 0; j < groups; j += 4) {
            const float4 q = *reinterpret_cast<const float4*>(tops + j);
            larger += (q.x > mine) + (q.y > mine) + (q.z > mine) + (q.w > mine);
            equal += (q.x == mine) + (q.y == mine) + (q.z == mine) + (q.w == mine);
        }
        if (larger < K && larger + equal >= K) s_bound = mine;
    }
    __syncthreads();
    const float bound = s_bound;
#pragma unroll
    for (int u = 0; u < BEAM_LOADS; ++u)
        if (column[u] >= bound && column[u] > -INFINITY) columns[atomicAdd(&s_columns, 1)] = (unsigned short)(u * BEAM_THREADS + tid);
    __syncthreads();
    // ---- their elements; after every 256 loads there is room for all that the next ones may bring
    const int tiles = (p1 - p0 + BEAM_TILE - 1) / BEAM_TILE, loads = s_columns * tiles;
    u64 least = 0ull;
    auto rank = [&](int n) {                // the K best of the n candidates into `sorted`, in order
        for (int i = tid; i < n; i += BEAM_THREADS) {
            const u64 mine = list[i];
            int better = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) better += list[j] > mine;
            if (better < K) sorted[better] = mine;
        }
        __syncthreads();
    };
    for (int l0 = 0; l0 < loads; l0 += BEAM_AGAIN * BEAM_THREADS) {
        float v[BEAM_AGAIN][4];
        int at[BEAM_AGAIN];
#pragma unroll
        for (int j = 0; j < BEAM_AGAIN; ++j) {
            const int l = l0 + j * BEAM_THREADS + tid, c = l / tiles;
            at[j] = l < loads ? p0 + (l - c * tiles) * BEAM_TILE + columns[c] * 4 : p1;
            if (VEC && at[j] + 4 <= p1) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(x + at[j]));
                v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = at[j] + e < p1 ? __ldg(x + at[j] + e) : -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < BEAM_AGAIN; ++j) {
            const int done = l0 + (j + 1) * BEAM_THREADS;
            if (done - BEAM_THREADS >= loads) break;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[j][e] >= bound && v[j][e] > -INFINITY) {
                    const u64 key = beam_key(v[j][e], at[j] + e);
                    if (key > least) list[atomicAdd(&s_n, 1)] = key;
                }
            __syncthreads();
            const int n = s_n;
            if (done < loads && n > BEAM_LIST - 4 * BEAM_THREADS) {
                rank(n);
                if (tid < K) list[tid] = sorted[tid];
                if (tid == 0) s_n = K;
                least = sorted[K - 1];
                __syncthreads();
            } else if (done < loads) {
                __syncthreads();            // all have read the number of candidates
            }
        }
    }
    rank(s_n);
    const size_t at = (size_t)r * gridDim.x + part;
    if (tid < K) best[at * K + tid] = sorted[tid];
    if (tid < 32) {
        const float2 q = tid < BEAM_THREADS / 32 ? warp_sums[tid] : make_float2(-INFINITY, 0.f);
        const float all = warp_max(q.x);
        const float total = warp_sum(q.x == -INFINITY ? q.y : q.y * beam_exp2((q.x - all) * LOG2E));
        if (tid == 0) sums[at] = make_float2(all, total);
    }
}

// A finite number as a whole one that is ordered as it and above 0 (-0 counts as 0), and back.
__device__ __forceinline__ u64 beam_order(double v) {
    const u64 bits = (u64)__double_as_longlong(v + 0.0);
    return bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}
__device__ __forceinline__ double beam_unorder(u64 o) { return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o)); }

// How many of the K numbers of a falling list are larger than x.
__device__ __forceinline__ int beam_count(const u64* list, int K, u64 x) {
    int lo = 0, hi = K;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}
// The lane with the largest of a warp's 64-bit numbers, of equal ones the first, as a bit; 0: all are 0 (others have higher halves above 0).  Mostly the higher
// halves tell; the chain of a round is a maximum, a vote and a branch that all lanes take alike (some 80 cycles).
__device__ __forceinline__ unsigned beam_winner(u64 v) {
    const unsigned hi = (unsigned)(v >> 32), top = __reduce_max_sync(0xffffffffu, hi);
    unsigned lanes = __ballot_sync(0xffffffffu, hi == top);
    if (lanes & (lanes - 1u)) {
        if (top == 0u) return 0u;
        const unsigned lo = hi == top ? (unsigned)v : 0u, low = __reduce_max_sync(0xffffffffu, lo);
        lanes = __ballot_sync(0xffffffffu, hi == top && lo == low);
        lanes &= 0u - lanes;
    }
    return lanes;
}

// Grid (groups).  First the lists of each row's parts become one: with many parts and few candidates (`rounds`) a warp takes a row, a lane each list, and the
// largest head is taken K times; else two neighbours at a time are merged, every key finding its place by searching the other list, so that a level
// costs a few dependent loads however long the lists are.  Then the first warp ranks the rows' lists against one another, a lane for each row,
// until B candidates that go on are found.  What a round waits for are the two warp-wide maxima and the winner's next number, which is there
// already.  The kernel is all latency.  One request of four beams: 6,500 cycles, of which loads and normalisers 2,000, merging 1,800, ranking 1,100.
__global__ void __launch_bounds__(1024) beam_join_kernel(const u64* __restrict__ best, const float2* __restrict__ sums, int parts, int K, int rows,
                                                         int beams, int end_token, bool rounds, const float* scores, int* tokens, int* parents,
                                                         float* out_scores, float* ended) {
    pdl_launch_dependents();
    __shared__ double offsets[BEAM_MAX], tops[BEAM_MAX];
    __shared__ int ends[BEAM_MAX];                              // which of a row's candidates is the end token
    __shared__ int taken[2 * BEAM_MAX];                         // which of its row's candidates has a rank
    extern __shared__ __align__(16) u64 beam_keys[];            // [rows * parts][K], and as many lists as half of the parts make
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int n = rows * parts * K;
    u64 *from = beam_keys, *to = from + n;
    pdl_wait();
    {
        const unsigned place = (unsigned)__cvta_generic_to_shared(from);
        const u64* source = best + (size_t)g * n;
#pragma unroll 1
        for (int i = tid; i < n; i += blockDim.x)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(place + 8u * i), "l"(source + i) : "memory");
    }
#pragma unroll 1
    for (int b = tid >> 5; b < rows; b += blockDim.x >> 5) {
        const size_t row = (size_t)g * rows + b;
        const float2 c = lane < parts ? sums[row * parts + lane] : make_float2(-INFINITY, 0.f);
        const float score = scores[row];
        const float top = warp_max(c.x);
        const float sum = warp_sum(c.x == -INFINITY ? c.y : c.y * beam_exp2((c.x - top) * 1.4426950408889634f));
        // log(f * 2^e), f in [1, 2): the whole part in 64 bits, so that the result is off by the rounding of a number below 0.7
        const int e = (int)(__float_as_uint(sum) >> 23) - 127;
        const float f = __uint_as_float((__float_as_uint(sum) & 0x007fffffu) | 0x3f800000u);
        // (a row with an infinity or without any number: its sum is none or 0)
        const bool dead = !(sum > 0.f && sum < INFINITY) || !isfinite(score);
        if (lane == 0) {
            // v = (x - largest) + (s - log sum): as near to s as it gets, however large the logits are
            offsets[b] = dead ? INFINITY : (double)score - ((double)e * 0.69314718055994530942 + (double)logf(f));
            tops[b] = (double)top;
            ends[b] = -1;
        }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    __syncthreads();
    int lists = parts;                  // of a row
    if (rounds) {
#pragma unroll 1
        for (int b = tid >> 5; b < rows; b += blockDim.x >> 5) {
            const u64* q = from + (b * parts + lane) * K;
            int k = 0;
            u64 head = lane < parts ? q[0] : 0ull, next = lane < parts && K > 1 ? q[1] : 0ull;
#pragma unroll 1
            for (int j = 0; j < K; ++j) {
                const unsigned winner = beam_winner(head);
                const bool won = (winner >> lane) & 1u;
                if (won || (winner == 0u && lane == 0)) to[b * K + j] = head;
                k += won;
                head = won ? next : head;
                next = lane < parts && k + 1 < K ? q[k + 1] : 0ull;
            }
        }
        from = to;
        __syncthreads();
    } else {
#pragma unroll 1
        while (lists > 1) {
            const int left = (lists + 1) >> 1;
#pragma unroll 1
            for (int i = tid; i < rows * lists * K; i += blockDim.x) {
                const int l = i / K, b = l / lists, p = l - b * lists, other = p ^ 1;
                const u64 x = from[i];
                int at = i - l * K;
                if (other < lists) at += beam_count(from + (l - p + other) * K, K, x);
                // (of empty places, which are equal, the odd list's come behind)
                if (x == 0ull && (p & 1)) at = K;
                if (at < K) to[(b * left + (p >> 1)) * K + at] = x;
            }
            __syncthreads();
            u64* const v = from;
            from = to;
            to = v;
            lists = left;
        }
    }
    // ---- keys become values, their tokens beside them
    int* const at = reinterpret_cast<int*>(beam_keys + n + (size_t)rows * ((parts + 1) / 2) * K);
#pragma unroll 1
    for (int i = tid; i < rows * K; i += blockDim.x) {
        const int b = i / K;
        const u64 key = from[i];
        const double off = offsets[b];
        from[i] = key && off < INFINITY ? beam_order(((double)beam_key_logit(key) - tops[b]) + off) : 0ull;
        at[i] = beam_key_at(key);
        if (key && beam_key_at(key) == end_token) ends[b] = i - b * K;
    }
    __syncthreads();
    if (tid >= 32) return;
    const int row = lane < rows ? lane : 0;
    const u64* list = from + row * K;
    const int end_at = lane < rows ? ends[lane] : -1;
    int k = 0;
    u64 value = lane < rows ? list[0] : 0ull, next = lane < rows && K > 1 ? list[1] : 0ull;
    int my_rank = -1, end_k = -1, count = 0;
    unsigned my_bit = 0u, has = 0u;     // the parent; parents with a child
    bool extra = lane < beams;
#pragma unroll 1
    for (int rank = 0; count < beams && rank < K; ++rank) {
        const unsigned at_end = __ballot_sync(0xffffffffu, k == end_at);
        const unsigned winner = beam_winner(value);             // of equal ones the first beam
        if (winner == 0u) break;
        const bool won = (winner >> lane) & 1u, ends_here = (at_end & winner) != 0u;
        if (won) taken[rank] = k;
        if (won && ends_here && rank < beams) end_k = k;
        if (lane == count && !ends_here) {
            my_rank = rank;
            my_bit = winner;
            extra = has & winner;
        }
        has |= ends_here ? 0u : winner;
        count += !ends_here;
        k += won;
        value = won ? next : value;
        next = lane < rows && k + 1 < K ? list[k + 1] : 0ull;
    }
    __syncwarp();
    const int my_parent = __ffs(my_bit) - 1, my_k = my_rank < 0 ? 0 : taken[my_rank];
    // places: the first child of a parent has the parent's, the others (and those that hold nothing) the ones that are left
    const unsigned others = __ballot_sync(0xffffffffu, extra);
    if (lane < beams) {
        int place = my_parent;
        if (extra) {
            unsigned left = (beams == 32 ? 0xffffffffu : (1u << beams) - 1u) & ~has;
            for (int e = __popc(others & ((1u << lane) - 1u)); e > 0; --e) left &= left - 1u;
            place = __ffs(left) - 1;
        }
        const int o = g * beams + place;
        tokens[o] = my_parent < 0 ? -1 : at[my_parent * K + my_k];
        parents[o] = my_parent < 0 ? place : my_parent;
        out_scores[o] = my_parent < 0 ? -INFINITY : (float)beam_unorder(from[my_parent * K + my_k]);
    }
    if (lane < rows) ended[g * rows + lane] = end_k < 0 ? -INFINITY : (float)beam_unorder(list[end_k]);
}

#define BEAM_JOIN_KEYS 8192     // candidates that a block of beam_join_kernel has room for in shared memory (with the merged ones and their tokens up to
                                // 108 KB: 28 rows of 29 beams in 5 parts)

// Parts of a row: as many as run at once over all rows (256 rows of 151,936 in 1 / 2 / 3 / 4 / 7 parts: 44 / 43 / 35 / 42 / 36 us with the join of then, now 32 in 3;
// four rows in 7 / 10 / 19: 8.9 / 8.3 / 7.6), none shorter than a tile, and no more than the join (a lane each) and the scratch have room for.
static int beam_parts(int groups, int rows, int V, int K, long long lists) {
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE, R = groups * rows;
    long long want = (6 * pico_num_sms()) / R;
    if (want > 32) want = 32;
    if (want > BEAM_JOIN_KEYS / (rows * K)) want = BEAM_JOIN_KEYS / (rows * K);
    if (want > lists / R) want = lists / R;
    const int parts = want < 1 ? 1 : want > tiles ? tiles : (int)want;
    const int each = (tiles + parts - 1) / parts;
    return (tiles + each - 1) / each;
}

// logits: [groups * rows, row_stride] float32, the first V columns are used; scores: [groups, rows].  tokens, parents, out_scores: [groups, beams];
// ended: [groups, rows].  end_token < 0: none.  out_scores may be scores where rows == beams.
// scratch: `lists` lists of 16 * beams + 8 bytes (8 * beams + 8 without an end token), from a 16-byte boundary on; one for each row at least, and 960 let
// rows be read in as many parts as a device of 160 multiprocessors runs at once.
PICO_API int pico_beam_select(const float* logits, long long row_stride, int groups, int rows, int V, int beams, int end_token, const float* scores,
                              void* scratch, int lists, int* tokens, int* parents, float* out_scores, float* ended, cudaStream_t stream) {
    if (groups < 1 || rows < 1 || rows > beams || beams > BEAM_MAX || V < 1 || (long long)groups * rows > 65535 ||
        (long long)rows * V > 0x7ff00000ll || lists < groups * rows)
        return PICO_ERR_SIZE;
    const int K = end_token >= 0 ? 2 * beams : beams, R = groups * rows, parts = beam_parts(groups, rows, V, K, lists);
    const int tiles = (V + BEAM_TILE - 1) / BEAM_TILE, per = (tiles + parts - 1) / parts * BEAM_TILE;
    int sets = 32;
    while (sets < 2 * K) sets *= 2;
    u64* best = reinterpret_cast<u64*>(scratch);
    float2* sums = reinterpret_cast<float2*>(best + (size_t)R * parts * K);
    const bool vec = row_stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    const int n = rows * parts * K;
    const size_t smem = (size_t)(n + rows * ((parts + 1) / 2) * K) * sizeof(u64) + (size_t)rows * K * sizeof(int);
    if (smem > 40 * 1024) {             // beside the kernel's own
        const cudaError_t e = pico_allow_smem<beam_join_kernel>(smem);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return (int)e;
        }
    }
    // a round takes some 100 cycles or more, as many warps as there are rows share the multiprocessor; a level of merging 350, or two a number (16 rows of 8
    // beams in 19 parts: by rounds 10.7 us, by levels 11.8; two of 28 beams in 16 parts 17.6 and 14.1)
    int by_rounds = K * (100 > 6 * rows ? 100 : 6 * rows), by_levels = 0;
    for (int left = parts, m = n; left > 1; left = (left + 1) / 2, m = rows * left * K) by_levels += 2 * m > 350 ? 2 * m : 350;
    const bool rounds = by_rounds < by_levels;
    int threads = ((rounds ? rows * K : n) / 2 + 31) / 32 * 32;
    threads = threads < 128 ? 128 : threads;
    threads = threads < 32 * rows ? 32 * rows : threads > 1024 ? 1024 : threads;
    pico_launch(vec ? beam_rows_kernel<true> : beam_rows_kernel<false>, dim3(parts, R), dim3(BEAM_THREADS), 0, stream, logits, row_stride, V, K, sets, per, best, sums);
    const int status = pico_launch_status();
    if (status) return status;
    pico_launch(beam_join_kernel, dim3(groups), dim3(threads), smem, stream, (const u64*)best, (const float2*)sums, parts, K, rows, beams, end_token,
                rounds, scores, tokens, parents, out_scores, ended);
    return pico_launch_status();
}
