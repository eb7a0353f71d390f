// Table rows looked up by number, and their gradient by sorted numbers.
//     out[i] = scale * table[id_i]  (negative id: an empty slot, zeros; id >= codes: NaN, so that the mistake shows)
//     dtable[v] = scale * sum_{i: id_i = v} dout[i]   - every element of dtable is written exactly once, zeros where no id points
// Forward is a copy: bound by the bytes of the output and of the rows it touches.
// Backward reads dout once and writes dtable once.  Atomic adds would make the sums depend on the order of arrival and would queue up on frequent numbers;
// here the positions are sorted by (id, position), a team of lanes adds P consecutive entries of the sorted list in fp32, and what a chunk boundary cuts
// is handed to the next level: a run of equal ids that lies inside one chunk is finished there, a run that reaches over an edge leaves a partial row in a
// list of at most two entries per chunk, which is a sorted list again and goes through the same kernel.  Work per team is P rows however
// the ids are distributed (one id 10^6 times: three more small levels), the order of every sum is fixed, and the result is the same in every run.
// Sorting: up to 4096 ids in one workgroup (bitonic, on (id, position) pairs, which are distinct); more: stable radix passes of up to 10 bits.
#include "stream_types.h"

namespace {

constexpr unsigned kEmpty = 0xffffffffu, kCarry = 0x80000000u;      // list keys: no entry; the run goes on here, but this entry has no row
constexpr int kSmall = 4096;                                        // ids sorted in one workgroup
constexpr int kChunk = 16384, kWaves = 16, kPerWave = kChunk / kWaves;
constexpr int kMaxBits = 10;

// sort key of an id: the id itself, `codes` (behind every table row) for ids that point nowhere
template <typename I> __device__ __forceinline__ unsigned key_of(const I* __restrict__ ids, int64_t i, int64_t codes) {
    const int64_t id = (int64_t)ids[i];
    return id < 0 || id >= codes ? (unsigned)codes : (unsigned)id;
}

// ---- forward -------------------------------------------------------------------------------------------------------------------------------
// A team of TEAM lanes per row, V values per lane and step; 4 rows per team so that four row reads are in flight.
template <typename T, typename O, typename I, int TEAM, int V>
__global__ __launch_bounds__(256) void lookup_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ table, O* __restrict__ out, int64_t n, int64_t codes, int dim, float scale) {
    constexpr int kTeams = 256 / TEAM, kRows = 4;
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const int64_t r0 = ((int64_t)blockIdx.x * kRows) * kTeams + team;
    int64_t id[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) id[r] = r0 + r * kTeams < n ? (int64_t)ids[r0 + r * kTeams] : -1;
    for (int c0 = lane * V; c0 < dim; c0 += TEAM * V) {
        const int c = min(c0, dim - V);                              // the last vector of an odd width is moved back: its first columns are written twice, with the same values
        float f[kRows][V];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const bool ok = id[r] >= 0 && id[r] < codes;
            if (ok) nvp_load<T, V>(table + id[r] * dim + c, f[r]);
#pragma unroll
            for (int e = 0; e < V; ++e) f[r][e] = ok ? f[r][e] * scale : id[r] < 0 ? 0.f : __uint_as_float(0x7fc00000u);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (r0 + r * kTeams < n) nvp_store<O, V>(out + (r0 + r * kTeams) * dim + c, f[r]);
    }
}

// ---- sorting -------------------------------------------------------------------------------------------------------------------------------
template <typename I>
__global__ __launch_bounds__(1024) void sort_small_kernel(const I* __restrict__ ids, unsigned* __restrict__ keys, unsigned* __restrict__ order, int n, int64_t codes, int padded) {
    __shared__ unsigned long long s[kSmall];
    for (int i = threadIdx.x; i < padded; i += 1024) s[i] = i < n ? (unsigned long long)key_of(ids, i, codes) << 32 | (unsigned)i : ~0ull;
    for (int size = 2; size <= padded; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < padded / 2; t += 1024) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const unsigned long long a = s[i], b = s[j];
                if ((a > b) == ((i & size) == 0)) {
                    s[i] = b;
                    s[j] = a;
                }
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 1024) {
        keys[i] = (unsigned)(s[i] >> 32);
        order[i] = (unsigned)s[i];
    }
}

// one radix pass in three launches: counts per (chunk, digit); exclusive prefix in (digit, chunk) order, by one workgroup; stable scatter
template <typename I, bool FIRST>
__global__ __launch_bounds__(1024) void radix_count_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys, unsigned* __restrict__ count, int64_t n, int64_t codes, int shift, int bits) {
    __shared__ unsigned bin[1 << kMaxBits];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += 1024) bin[b] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kChunk;
    for (int j = 0; j < kChunk / 1024; ++j) {
        const int64_t i = base + j * 1024 + threadIdx.x;
        if (i < n) atomicAdd(&bin[((FIRST ? key_of(ids, i, codes) : keys[i]) >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 1024) count[(int64_t)blockIdx.x * bins + b] = bin[b];
}

__global__ __launch_bounds__(1024) void radix_scan_kernel(unsigned* __restrict__ count, int chunks, int bits) {
    __shared__ unsigned wsum[16];
    const int bins = 1 << bits, b = threadIdx.x;
    unsigned sum = 0u;
    if (b < bins)
        for (int c = 0; c < chunks; ++c) sum += count[(int64_t)c * bins + b];
    unsigned inc = sum;                                              // inclusive prefix over the digits: within the wave, then over the waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(inc, o);
        if ((threadIdx.x & 63) >= o) inc += up;
    }
    if ((threadIdx.x & 63) == 63) wsum[threadIdx.x >> 6] = inc;
    __syncthreads();
    unsigned run = inc - sum;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) run += wsum[w];
    if (b < bins)
        for (int c = 0; c < chunks; ++c) {
            const unsigned v = count[(int64_t)c * bins + b];
            count[(int64_t)c * bins + b] = run;
            run += v;
        }
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(1024) void radix_scatter_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys, const unsigned* __restrict__ pos, const unsigned* __restrict__ count,
                                                             unsigned* __restrict__ keys_out, unsigned* __restrict__ pos_out, int64_t n, int64_t codes, int shift, int bits) {
    extern __shared__ unsigned cursor[];                             // [16 waves][bins]
    const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = threadIdx.x; b < kWaves * bins; b += 1024) cursor[b] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kChunk + (int64_t)wave * kPerWave;      // a wave's ids are consecutive: waves in order, rounds in order, lanes in order
    unsigned k[kPerWave / 64];
#pragma unroll
    for (int j = 0; j < kPerWave / 64; ++j) {
        const int64_t i = base + j * 64 + lane;
        k[j] = i < n ? (FIRST ? key_of(ids, i, codes) : keys[i]) : 0u;
        if (i < n) atomicAdd(&cursor[wave * bins + ((k[j] >> shift) & (bins - 1))], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 1024) {
        unsigned run = count[(int64_t)blockIdx.x * bins + b];
        for (int w = 0; w < kWaves; ++w) {
            const unsigned v = cursor[w * bins + b];
            cursor[w * bins + b] = run;
            run += v;
        }
    }
    __syncthreads();
    const unsigned long long below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
#pragma unroll
    for (int j = 0; j < kPerWave / 64; ++j) {
        const int64_t i = base + j * 64 + lane;
        const unsigned d = (k[j] >> shift) & (bins - 1);
        unsigned long long same = __ballot(i < n);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long m = __ballot((d >> b) & 1u);
            same &= ((d >> b) & 1u) ? m : ~m;
        }
        if (i < n) {
            const unsigned at = cursor[wave * bins + d] + (unsigned)__popcll(same & below);
            keys_out[at] = k[j];
            pos_out[at] = FIRST ? (unsigned)i : pos[i];
            if ((same >> lane) == 1ull) cursor[wave * bins + d] = at + 1u;       // the last of the equals moves the cursor; every lane has read it (one wave, in order)
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- sums over the sorted list ----------------------------------------------------------------------------------------------------------------
// Entry i of a list: keys[i] (kEmpty: none; | kCarry: no row) and a row of D values: dout row order[i] (first level) or partial row i.
// blocks < sum_blocks: a team of TEAM lanes adds P entries over TEAM * V columns (blockIdx.y: which columns).  The other blocks (first level only): zeros into
// the table rows no id points to, 64 rows per wave: every lane looks its row up in the sorted keys (binary search), the wave then writes the empty ones.
template <typename S, typename T, bool FIRST, int TEAM, int V, int BATCH>
__global__ __launch_bounds__(256) void sum_runs_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ order, const S* __restrict__ rows, T* __restrict__ dtable,
                                                       unsigned* __restrict__ next_keys, float* __restrict__ next_rows, int64_t m, int per_chunk, int64_t chunks, int64_t sum_blocks, int64_t codes,
                                                       int dim, float scale) {
    constexpr int kTeams = 256 / TEAM;
    if (FIRST && (int64_t)blockIdx.x >= sum_blocks) {
        const int lane = threadIdx.x & 63;
        const int64_t r0 = (((int64_t)blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * 64;
        const int64_t row = r0 + lane;
        bool empty = false;
        if (row < codes) {
            int64_t lo = 0, hi = m;
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (keys[mid] < (unsigned)row) lo = mid + 1;
                else hi = mid;
            }
            empty = lo >= m || keys[lo] != (unsigned)row;
        }
        unsigned long long todo = __ballot(empty);
        const float zero[V] = {};
        const int c0 = blockIdx.y * (TEAM * V), cw = min(TEAM * V, dim - c0);
        while (todo) {
            const int64_t at = r0 + __ffsll((long long)todo) - 1;
            todo &= todo - 1;
            for (int c = lane * V; c < cw; c += 64 * V) nvp_store<T, V>(dtable + at * dim + min(c0 + c, dim - V), zero);
        }
        return;
    }
    const int lane = threadIdx.x % TEAM;
    const int64_t ch = (int64_t)blockIdx.x * kTeams + threadIdx.x / TEAM;
    if (ch >= chunks) return;
    const bool live = (blockIdx.y * TEAM + lane) * V < dim;
    const int c = min((int)(blockIdx.y * TEAM + lane) * V, dim - V);      // the last vector of an odd width is moved back: its first columns are summed and written twice, alike
    const int64_t lo = ch * per_chunk, hi = min(lo + per_chunk, m);
    const unsigned before = lo > 0 ? keys[lo - 1] : kEmpty, after = hi < m ? keys[hi] : kEmpty;
    unsigned cur = kEmpty, head_key = kEmpty, tail_key = kEmpty;
    bool from_left = false;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    const auto same_run = [](unsigned a, unsigned b) { return a != kEmpty && b != kEmpty && ((a ^ b) & ~kCarry) == 0u; };
    // the run in `cur` is over: `to_right` says that it goes on in the next chunk
    const auto flush = [&](bool to_right) {
        if (cur == kEmpty) return;
        if (!from_left && !to_right) {
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = acc[e] * scale;
            if (live) nvp_store<T, V>(dtable + (int64_t)cur * dim + c, f);
        } else {
            const int64_t slot = 2 * ch + (from_left ? 0 : 1);
            if (live) nvp_store<float, V>(next_rows + slot * dim + c, acc);
            if (from_left) head_key = cur;
            else tail_key = cur;
            if (from_left && to_right) tail_key = cur | kCarry;       // the whole chunk is inside one run: one row, and a key that keeps the run together
        }
    };
    for (int64_t i0 = lo; i0 < hi; i0 += BATCH) {
        unsigned k[BATCH];
        float f[BATCH][V];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int64_t i = i0 + b;
            k[b] = i < hi ? keys[i] : kEmpty;
            if (FIRST && k[b] >= (unsigned)codes) k[b] = kEmpty;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int64_t i = i0 + b;
            const bool has = live && k[b] != kEmpty && !(k[b] & kCarry);
            const int64_t src = has ? (FIRST ? (int64_t)order[i] : i) : 0;
            if (has) nvp_load<S, V>(rows + src * dim + c, f[b]);
#pragma unroll
            for (int e = 0; e < V; ++e) f[b][e] = has ? f[b][e] : 0.f;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            if (k[b] == kEmpty) continue;
            const unsigned key = k[b] & ~kCarry;
            if (key != cur) {
                flush(false);
                from_left = i0 + b == lo && same_run(before, key);
                cur = key;
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += f[b][e];
        }
    }
    flush(same_run(cur, after));
    if (next_keys && lane == 0 && blockIdx.y == 0) {
        next_keys[2 * ch] = head_key;
        next_keys[2 * ch + 1] = tail_key;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------
int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }
constexpr int kPerChunk1 = 32, kPerChunk2 = 64;

struct Plan {
    bool small;
    int passes, bits;
    int64_t radix_chunks;
    int per_chunk;                  // first level
    int levels;
    int64_t m[12], chunks[12];      // entries and chunks of each level
    int64_t off_key[2], off_pos[2], off_count, off_lkey[2], off_lrow[2], bytes;
};
Plan plan_of(int64_t n, int64_t codes, int64_t dim) {
    Plan P{};
    P.small = n <= kSmall;
    int b = 1;
    while (b < 32 && ((codes + 1) - 1) >> b) ++b;                    // keys 0 .. codes
    P.passes = (b + kMaxBits - 1) / kMaxBits;
    P.bits = (b + P.passes - 1) / P.passes;
    P.radix_chunks = (n + kChunk - 1) / kChunk;
    P.per_chunk = n < 65536 ? 16 : kPerChunk1;                       // short lists: more teams with less to do one after another
    int64_t m = n;
    for (P.levels = 0;;) {
        const int per = P.levels == 0 ? P.per_chunk : kPerChunk2;
        P.m[P.levels] = m;
        P.chunks[P.levels] = (m + per - 1) / per;
        const bool done = P.chunks[P.levels] <= 1;
        m = 2 * P.chunks[P.levels];
        ++P.levels;
        if (done) break;
    }
    int64_t at = 0;
    for (int i = 0; i < (P.small ? 1 : 2); ++i) {
        P.off_key[i] = at;
        at += up256(n * 4);
        P.off_pos[i] = at;
        at += up256(n * 4);
    }
    P.off_count = at;
    if (!P.small) at += up256(P.radix_chunks * (1ll << P.bits) * 4);
    for (int i = 0; i < 2; ++i) {                                    // level l writes list l & 1: a later list is never longer than the one it replaces
        const int64_t e = i + 1 < P.levels ? P.m[i + 1] : 0;
        P.off_lkey[i] = at;
        at += up256(e * 4);
        P.off_lrow[i] = at;
        at += up256(e * dim * 4);
    }
    P.bytes = at;
    return P;
}

int bad_sizes(int64_t n, int64_t codes, int64_t dim) {
    if (n < 0 || codes < 1 || dim < 1) return NVP_ERR_BADARG;
    return n > (1ll << 31) - 1 || codes > (1ll << 31) - 2 || dim > (1 << 24) ? NVP_ERR_UNSUPPORTED : 0;
}
// 16-byte accesses of the narrower of two types
template <typename A, typename B> constexpr int vec_of() { return 16 / (sizeof(A) > sizeof(B) ? sizeof(A) : sizeof(B)); }

int team_of(int64_t lanes) { return lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64; }

template <typename T, typename O, typename I, int V>
int fwd(const I* ids, const T* table, O* out, int64_t n, int64_t codes, int dim, float scale, hipStream_t st) {
    const int team = team_of((dim + V - 1) / V);
    const int64_t blocks = (n + 4 * (256 / team) - 1) / (4 * (256 / team));
    if (blocks > 0x7fffffff) return NVP_ERR_UNSUPPORTED;
    const dim3 g((unsigned)blocks), wg(256);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, wg, 0, st, ids, table, out, n, codes, dim, scale); };
    if (team == 4) go(lookup_fwd_kernel<T, O, I, 4, V>);
    else if (team == 8) go(lookup_fwd_kernel<T, O, I, 8, V>);
    else if (team == 16) go(lookup_fwd_kernel<T, O, I, 16, V>);
    else if (team == 32) go(lookup_fwd_kernel<T, O, I, 32, V>);
    else go(lookup_fwd_kernel<T, O, I, 64, V>);
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename S, typename T, bool FIRST, int V>
int sum_level(const unsigned* keys, const unsigned* order, const S* rows, T* dtable, unsigned* nkeys, float* nrows, int64_t m, int per_chunk, int64_t chunks, int64_t codes, int dim, float scale,
              hipStream_t st) {
    const int team = team_of((dim + V - 1) / V), teams = 256 / team;
    const int64_t sums = (chunks + teams - 1) / teams, fill = FIRST ? (codes + 255) / 256 : 0, cols = (dim + team * V - 1) / (team * V);
    if (sums + fill > 0x7fffffff || cols > 65535) return NVP_ERR_UNSUPPORTED;
    const dim3 g((unsigned)(sums + fill), (unsigned)cols), wg(256);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, wg, 0, st, keys, order, rows, dtable, nkeys, nrows, m, per_chunk, chunks, sums, codes, dim, scale); };
    if (team == 4) go(sum_runs_kernel<S, T, FIRST, 4, V, 8>);
    else if (team == 8) go(sum_runs_kernel<S, T, FIRST, 8, V, 8>);
    else if (team == 16) go(sum_runs_kernel<S, T, FIRST, 16, V, 8>);
    else if (team == 32) go(sum_runs_kernel<S, T, FIRST, 32, V, 8>);
    else go(sum_runs_kernel<S, T, FIRST, 64, V, 8>);
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename S, typename T, int V, int VF>
int sums(const Plan& P, const unsigned* keys, const unsigned* order, const S* dout, T* dtable, uint8_t* ws, int64_t codes, int dim, float scale, hipStream_t st) {
    const auto lkey = [&](int l) { return (unsigned*)(ws + P.off_lkey[l & 1]); };
    const auto lrow = [&](int l) { return (float*)(ws + P.off_lrow[l & 1]); };
    const bool more = P.levels > 1;
    int rc = sum_level<S, T, true, V>(keys, order, dout, dtable, more ? lkey(0) : nullptr, more ? lrow(0) : nullptr, P.m[0], P.per_chunk, P.chunks[0], codes, dim, scale, st);
    for (int l = 1; !rc && l < P.levels; ++l) {
        const bool next = l + 1 < P.levels;
        rc = sum_level<float, T, false, VF>(lkey(l - 1), nullptr, lrow(l - 1), dtable, next ? lkey(l) : nullptr, next ? lrow(l) : nullptr, P.m[l], kPerChunk2, P.chunks[l], codes, dim, scale, st);
    }
    return rc;
}

template <typename I, typename S, typename T>
int bwd(const I* ids, const S* dout, T* dtable, int64_t n, int64_t codes, int dim, float scale, uint8_t* ws, hipStream_t st) {
    const Plan P = plan_of(n, codes, dim);
    unsigned *key[2], *pos[2];
    for (int i = 0; i < 2; ++i) {
        key[i] = (unsigned*)(ws + P.off_key[P.small ? 0 : i]);
        pos[i] = (unsigned*)(ws + P.off_pos[P.small ? 0 : i]);
    }
    int at = 0;
    if (n == 0) {
        // nothing to sort: the sums below only write zeros
    } else if (P.small) {
        int padded = 2;
        while (padded < n) padded <<= 1;
        hipLaunchKernelGGL((sort_small_kernel<I>), dim3(1), dim3(1024), 0, st, ids, key[0], pos[0], (int)n, codes, padded);
        NVP_LAUNCH_CHECK();
    } else {
        unsigned* count = (unsigned*)(ws + P.off_count);
        const dim3 g((unsigned)P.radix_chunks), wg(1024);
        const size_t lds = (size_t)kWaves * (1u << P.bits) * 4;
        for (int p = 0; p < P.passes; ++p) {
            const int shift = p * P.bits;
            const unsigned *kin = key[at], *pin = pos[at];
            unsigned *kout = key[at ^ 1], *pout = pos[at ^ 1];
            if (p == 0) hipLaunchKernelGGL((radix_count_kernel<I, true>), g, wg, 0, st, ids, kin, count, n, codes, shift, P.bits);
            else hipLaunchKernelGGL((radix_count_kernel<I, false>), g, wg, 0, st, ids, kin, count, n, codes, shift, P.bits);
            NVP_LAUNCH_CHECK();
            hipLaunchKernelGGL(radix_scan_kernel, dim3(1), wg, 0, st, count, (int)P.radix_chunks, P.bits);
            NVP_LAUNCH_CHECK();
            if (p == 0) hipLaunchKernelGGL((radix_scatter_kernel<I, true>), g, wg, lds, st, ids, kin, pin, count, kout, pout, n, codes, shift, P.bits);
            else hipLaunchKernelGGL((radix_scatter_kernel<I, false>), g, wg, lds, st, ids, kin, pin, count, kout, pout, n, codes, shift, P.bits);
            NVP_LAUNCH_CHECK();
            at ^= 1;
        }
    }
    constexpr int V = vec_of<S, T>();
    if (dim >= (V > 4 ? V : 4)) return sums<S, T, V, 4>(P, key[at], pos[at], dout, dtable, ws, codes, dim, scale, st);
    return sums<S, T, 1, 1>(P, key[at], pos[at], dout, dtable, ws, codes, dim, scale, st);
}

template <typename T, typename O>
int any_ids(const void* ids, int ids64, const void* a, void* b, bool backward, int64_t n, int64_t codes, int dim, float scale, uint8_t* ws, hipStream_t st) {
    if (backward) return ids64 ? bwd<int64_t, O, T>((const int64_t*)ids, (const O*)a, (T*)b, n, codes, dim, scale, ws, st) : bwd<int32_t, O, T>((const int32_t*)ids, (const O*)a, (T*)b, n, codes, dim, scale, ws, st);
    constexpr int V = vec_of<T, O>();
    const bool vec = dim >= V;
    if (ids64) return vec ? fwd<T, O, int64_t, V>((const int64_t*)ids, (const T*)a, (O*)b, n, codes, dim, scale, st) : fwd<T, O, int64_t, 1>((const int64_t*)ids, (const T*)a, (O*)b, n, codes, dim, scale, st);
    return vec ? fwd<T, O, int32_t, V>((const int32_t*)ids, (const T*)a, (O*)b, n, codes, dim, scale, st) : fwd<T, O, int32_t, 1>((const int32_t*)ids, (const T*)a, (O*)b, n, codes, dim, scale, st);
}
// table types: fp32 with any output type, or 16 bits with the same output type
int any_type(int32_t table_type, int32_t out_type, const void* ids, int ids64, const void* a, void* b, bool backward, int64_t n, int64_t codes, int dim, float scale, uint8_t* ws, hipStream_t st) {
    if (table_type == NVP_F32 && out_type == NVP_F32) return any_ids<float, float>(ids, ids64, a, b, backward, n, codes, dim, scale, ws, st);
    if (table_type == NVP_F32 && out_type == NVP_BF16) return any_ids<float, nvp_bf16>(ids, ids64, a, b, backward, n, codes, dim, scale, ws, st);
    if (table_type == NVP_F32 && out_type == NVP_F16) return any_ids<float, nvp_f16>(ids, ids64, a, b, backward, n, codes, dim, scale, ws, st);
    if (table_type == NVP_BF16 && out_type == NVP_BF16) return any_ids<nvp_bf16, nvp_bf16>(ids, ids64, a, b, backward, n, codes, dim, scale, ws, st);
    if (table_type == NVP_F16 && out_type == NVP_F16) return any_ids<nvp_f16, nvp_f16>(ids, ids64, a, b, backward, n, codes, dim, scale, ws, st);
    return NVP_ERR_BADARG;
}

}  // namespace

extern "C" int nvp_lookup_fwd(const void* ids, int32_t ids64, const void* table, int32_t table_type, void* out, int32_t out_type, int64_t n, int64_t codes, int64_t dim, float scale, void* stream) {
    const int rc = bad_sizes(n, codes, dim);
    if (rc) return rc;
    if (n == 0) return 0;
    if (!ids || !table || !out) return NVP_ERR_BADARG;
    return any_type(table_type, out_type, ids, ids64, table, out, false, n, codes, (int)dim, scale, nullptr, (hipStream_t)stream);
}

extern "C" int64_t nvp_lookup_bwd_workspace_bytes(int64_t n, int64_t codes, int64_t dim) {
    const int rc = bad_sizes(n, codes, dim);
    return rc ? rc : plan_of(n, codes, dim).bytes;
}

extern "C" int nvp_lookup_bwd(const void* ids, int32_t ids64, const void* dout, int32_t out_type, void* dtable, int32_t table_type, int64_t n, int64_t codes, int64_t dim, float scale,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = bad_sizes(n, codes, dim);
    if (rc) return rc;
    if (!dtable || (n && (!ids || !dout || !workspace || workspace_bytes < plan_of(n, codes, dim).bytes || ((uintptr_t)workspace & 15)))) return NVP_ERR_BADARG;
    return any_type(table_type, out_type, ids, ids64, dout, dtable, true, n, codes, (int)dim, scale, (uint8_t*)workspace, (hipStream_t)stream);
}
