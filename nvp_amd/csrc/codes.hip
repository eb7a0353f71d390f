// Table rows looked up by number, and their gradient by sorted numbers.
//     out[i] = scale * table[id_i]  (negative id: an empty slot, zeros; id >= codes: NaN, so that the mistake shows)
//     dtable[v] = scale * sum_{i: id_i = v} dout[i]   - every element of dtable is written exactly once, zeros where no id points
// Forward is a copy: bound by the bytes of the output and of the rows it touches.
// Backward reads dout once and writes dtable once.  Atomic adds would make the sums depend on the order of arrival and would queue up on frequent numbers;
// here the positions are sorted by (id, position), a team of lanes adds P consecutive entries of the sorted list in fp32, and what a chunk boundary cuts
// is handed to the next level: a run of equal ids that lies inside one chunk is finished there, a run that reaches over an edge leaves a partial row in a
// list of at most two entries per chunk, which is a sorted list again and goes through the same kernel.  Work per team is P rows however
// the ids are distributed (one id 10^6 times: three more small levels), the order of every sum is fixed, and the result is the same in every run.
// Sorting: up to 1024 ids in one workgroup (bitonic, on (id, position) pairs, which are distinct); more: stable radix passes of up to 10 bits.  Where codes are
// few and rows are narrow the batch is not sorted as a whole but chunk by chunk (further down).
#include <type_traits>
#include "stream_types.h"

namespace {

constexpr unsigned kEmpty = 0xffffffffu, kCarry = 0x80000000u;      // list keys: no entry; the run goes on here, but this entry has no row
constexpr int kSmall = 1024;                                        // ids sorted in one workgroup (1000 ids, us, so / by radix passes: 23 / 20 for one pass, 24 / 30 for two; 4096: 45 / 21, 49 / 34)
constexpr int kChunk = 2048, kWaves = 8, kPerWave = kChunk / kWaves; // ids per workgroup of a radix pass
constexpr int kMaxBits = 10;

// sort key of an id: the id itself, `codes` (behind every table row) for ids that point nowhere
template <typename I> __device__ __forceinline__ unsigned key_of(const I* __restrict__ ids, int64_t i, int64_t codes) {
    const int64_t id = (int64_t)ids[i];
    return id < 0 || id >= codes ? (unsigned)codes : (unsigned)id;
}

// ---- forward -------------------------------------------------------------------------------------------------------------------------------
// A team of TEAM lanes per row, V values per lane and step; 4 rows per team so that four row reads are in flight.  Bound by the writes of the output:
// 1 245 184 rows of 32 fp32 out of 600 take 29 us (169 MB written and read: 5.8 TB/s), 200 003 of 512 bf16 out of 50 000 55 us (256 MB, 4.65 TB/s;
// a large copy reaches 4.8 TB/s here, a fill 6.75).
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
// A short list of ids keeps few CUs busy: where most rows of the gradient stay empty the other workgroups of the sort's launches write zeros, each launch a part
// of the table.  Workgroups from `work` on write 64 KB each.
struct Fill {
    uint8_t* to;
    int64_t bytes;
    unsigned work;
};
constexpr int64_t kFillBytes = 65536;
__device__ __forceinline__ bool fills(const Fill& F) {
    if (blockIdx.x < F.work) return false;
    uint8_t* const to = F.to + (int64_t)(blockIdx.x - F.work) * kFillBytes;
    const int len = (int)min(kFillBytes, F.bytes - (int64_t)(blockIdx.x - F.work) * kFillBytes);
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x * 16; i + 16 <= len; i += blockDim.x * 16) nvp_store<float, 4>(reinterpret_cast<float*>(to + i), zero);
    for (int i = (len & ~15) + threadIdx.x; i < len; i += blockDim.x) to[i] = 0;
    return true;
}

template <typename I>
__global__ __launch_bounds__(1024) void sort_small_kernel(const I* __restrict__ ids, uint2* __restrict__ sorted, int n, int64_t codes, int padded, Fill fill) {
    __shared__ unsigned long long s[kSmall];
    if (fills(fill)) return;
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
    for (int i = threadIdx.x; i < n; i += 1024) sorted[i] = make_uint2((unsigned)(s[i] >> 32), (unsigned)s[i]);
}

// One radix pass in three launches: counts per (chunk, digit); per digit, the number of its ids in earlier chunks, and its total; stable scatter, where every
// workgroup adds up the totals of the smaller digits by itself.  A chunk is 2048 ids: its scatter goes through LDS, so that equal digits leave it side by side.
// Bound by latency, not bytes: a pass over 16 384 ids takes 3 + 3.5 + 7 us, over 200 003 ids 4.5 + 4.5 + 7 us.
template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void radix_count_kernel(const I* __restrict__ ids, const uint2* __restrict__ in, unsigned* __restrict__ count, int64_t n, int64_t codes, int shift, int bits,
                                                          Fill fill) {
    __shared__ unsigned bin[1 << kMaxBits];
    if (fills(fill)) return;
    const int bins = 1 << bits;
    const int64_t base = (int64_t)blockIdx.x * kChunk + threadIdx.x;
    unsigned k[kChunk / 256];
#pragma unroll
    for (int j = 0; j < kChunk / 256; ++j) k[j] = base + j * 256 < n ? (FIRST ? key_of(ids, base + j * 256, codes) : in[base + j * 256].x) : 0u;
    for (int b = threadIdx.x; b < bins; b += 256) bin[b] = 0u;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kChunk / 256; ++j)
        if (base + j * 256 < n) atomicAdd(&bin[(k[j] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) count[(int64_t)blockIdx.x * bins + b] = bin[b];
}

// count [chunk][digit] -> exclusive prefix over the chunks, total [digit].  A workgroup: 16 digits (lanes) x 64 spans of chunks: a span of 608 chunks
// (1.2 million ids) is 10 reads long, two waits for memory (64 digits x 16 spans: five, 9.6 against 5 us).
__global__ __launch_bounds__(1024) void radix_scan_kernel(unsigned* __restrict__ count, unsigned* __restrict__ total, int chunks, int bits, Fill fill) {
    __shared__ unsigned span[64][16], group[4][16];
    if (fills(fill)) return;
    const int bins = 1 << bits, digit = threadIdx.x & 15, s = threadIdx.x >> 4, b = blockIdx.x * 16 + digit;
    const int per = (chunks + 63) / 64, c0 = min(s * per, chunks), c1 = min(c0 + per, chunks);
    unsigned sum = 0u;
    if (b < bins)
        for (int c = c0; c < c1; c += 8) {
            unsigned t[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = c + k < c1 ? count[(int64_t)(c + k) * bins + b] : 0u;
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += t[k];
        }
    span[s][digit] = sum;
    __syncthreads();
    if (s < 4) {
        unsigned g = 0u;
#pragma unroll
        for (int w = 0; w < 16; ++w) g += span[s * 16 + w][digit];
        group[s][digit] = g;
    }
    __syncthreads();
    if (b >= bins) return;
    unsigned run = 0u;
    for (int w = 0; w < s >> 4; ++w) run += group[w][digit];
    for (int w = s & ~15; w < s; ++w) run += span[w][digit];
    if (s == 63) total[b] = run + sum;
    for (int c = c0; c < c1; c += 8) {
        unsigned t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = c + k < c1 ? count[(int64_t)(c + k) * bins + b] : 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k < c1) {
                count[(int64_t)(c + k) * bins + b] = run;
                run += t[k];
            }
    }
}

// Stable places by digit for a wave's ids, one round of 64 in turn: an id's place is its digit's cursor plus the number of equal digits in lanes before it, and the
// last of the equals moves the cursor (every lane has read it: one wave, in order).  `put` gets the round and the place.
template <int ROUNDS, typename P> __device__ __forceinline__ void place_ids(const unsigned (&d)[ROUNDS], int64_t base, int64_t n, int bits, unsigned* cursor, const P& put) {
    const int lane = threadIdx.x & 63;
    const unsigned long long below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
        const int64_t i = base + j * 64 + lane;
        if (base + j * 64 >= n) break;                                           // the wave's ids are over
        unsigned long long same = __ballot(i < n);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long m = __ballot((d[j] >> b) & 1u);
            same &= ((d[j] >> b) & 1u) ? m : ~m;
        }
        if (i < n) {
            const unsigned at = cursor[d[j]] + (unsigned)__popcll(same & below);
            put(j, at);
            if ((same >> lane) == 1ull) cursor[d[j]] = at + 1u;
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");                   // the next round reads what this one wrote (no instruction: LDS keeps a wave's order)
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(64 * kWaves) void radix_scatter_kernel(const I* __restrict__ ids, const uint2* __restrict__ in, const unsigned* __restrict__ count,
                                                            const unsigned* __restrict__ total, uint2* __restrict__ sorted, int64_t n, int64_t codes, int shift, int bits,
                                                            Fill fill) {
    __shared__ unsigned cursor[kWaves][1 << kMaxBits];                           // where the wave's next id of a digit goes in `list`
    __shared__ unsigned shift_to[1 << kMaxBits];                                 // place in the output - place in `list`, per digit
    __shared__ uint2 list[kChunk];
    __shared__ unsigned wsum[2][kWaves];
    if (fills(fill)) return;
    const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t base = (int64_t)blockIdx.x * kChunk + (int64_t)wave * kPerWave;      // a wave's ids are consecutive: waves in order, rounds in order, lanes in order
    constexpr int kRounds = kPerWave / 64, kPer = (1 << kMaxBits) / (64 * kWaves);
    unsigned k[kRounds], p[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
        const int64_t i = base + j * 64 + lane;
        if (FIRST) {
            k[j] = i < n ? key_of(ids, i, codes) : 0u;
            p[j] = (unsigned)i;
        } else {
            const uint2 t = i < n ? in[i] : make_uint2(0u, 0u);
            k[j] = t.x;
            p[j] = t.y;
        }
    }
    unsigned all[kPer], before[kPer], mine[kPer], sum[2] = {0u, 0u};             // a thread's digits: total, number in earlier chunks, number in this one
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int b = threadIdx.x * kPer + e;
        all[e] = b < bins ? total[b] : 0u;
        before[e] = b < bins ? count[(int64_t)blockIdx.x * bins + b] : 0u;
    }
    for (int b = threadIdx.x; b < kWaves << kMaxBits; b += 64 * kWaves) (&cursor[0][0])[b] = 0u;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRounds; ++j)
        if (base + j * 64 + lane < n) atomicAdd(&cursor[wave][(k[j] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    // where the digits start in the output (the totals of all smaller digits + the chunk's place among the chunks) and in this chunk
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int b = threadIdx.x * kPer + e;
        mine[e] = 0u;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mine[e] += cursor[w][b];
        sum[0] += all[e];
        sum[1] += mine[e];
    }
    unsigned inc[2] = {sum[0], sum[1]};
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const unsigned up = __shfl_up(inc[q], o);
            if (lane >= o) inc[q] += up;
        }
    if (lane == 63) {
        wsum[0][wave] = inc[0];
        wsum[1][wave] = inc[1];
    }
    __syncthreads();
    unsigned out = inc[0] - sum[0], here = inc[1] - sum[1];
    for (int w = 0; w < wave; ++w) {
        out += wsum[0][w];
        here += wsum[1][w];
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int b = threadIdx.x * kPer + e;
        if (b >= bins) break;
        shift_to[b] = out + before[e] - here;
        unsigned run = here;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const unsigned v = cursor[w][b];
            cursor[w][b] = run;
            run += v;
        }
        out += all[e];
        here += mine[e];
    }
    __syncthreads();
    unsigned d[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) d[j] = (k[j] >> shift) & (bins - 1);
    place_ids<kRounds>(d, base, n, bits, cursor[wave], [&](int j, unsigned at) { list[at] = make_uint2(k[j], p[j]); });
    __syncthreads();
    // equal digits lie side by side now: their places in the output do too, and neighbouring lanes write them together
    const int len = (int)min((int64_t)kChunk, n - (int64_t)blockIdx.x * kChunk);
    for (int t = threadIdx.x; t < len; t += 64 * kWaves) {
        const uint2 v = list[t];
        sorted[t + shift_to[(v.x >> shift) & (bins - 1)]] = v;
    }
}

// ---- sums over the sorted list ----------------------------------------------------------------------------------------------------------------
// Entry i of a list: a key (kEmpty: none; | kCarry: no row) and a row of D values.  First level: sorted (id, position) pairs, the row is dout row `position`;
// later: keys[i], partial row i.
// Bound by the bytes of dout, read in rows at the sorted positions, and of the table: 200 003 of 512 bf16 into 50 000 73 us (256 MB, 3.5 TB/s),
// 16 384 of 1024 bf16 into 65 536 fp32 rows 16 - 18 us (the empty rows are written beside the sort there, 268 MB in 55 us).
// blocks < sum_blocks: a team of TEAM lanes adds P entries over TEAM * V columns (blockIdx.y: which columns).  The other blocks (first level only): zeros into
// the table rows no id points to, 64 rows per wave: every lane looks its row up in the sorted keys (binary search), the wave then writes the empty ones.
template <typename S, typename T, bool FIRST, int TEAM, int V>
__global__ __launch_bounds__(256) void sum_runs_kernel(const uint2* __restrict__ sorted, const unsigned* __restrict__ keys, const S* __restrict__ rows, T* __restrict__ dtable,
                                                       unsigned* __restrict__ next_keys, float* __restrict__ next_rows, int64_t m, int per_chunk, int64_t chunks, int64_t sum_blocks, int64_t codes,
                                                       int dim, float scale) {
    constexpr int kTeams = 256 / TEAM, kBatch = V > 4 ? 8 : 16;      // rows in flight per team: 64 registers
    if (FIRST && (int64_t)blockIdx.x >= sum_blocks) {
        const int lane = threadIdx.x & 63;
        const int64_t r0 = (((int64_t)blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * 64;
        const int64_t row = r0 + lane;
        bool empty = false;
        if (row < codes) {
            int64_t lo = 0, hi = m;
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if (sorted[mid].x < (unsigned)row) lo = mid + 1;
                else hi = mid;
            }
            empty = lo >= m || sorted[lo].x != (unsigned)row;
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
    const int64_t lo = ch * per_chunk;
    const int len = (int)min((int64_t)per_chunk, m - lo);
    const auto key_at = [&](int64_t i) { return FIRST ? sorted[i].x : keys[i]; };
    const unsigned before = lo > 0 ? key_at(lo - 1) : kEmpty, after = lo + len < m ? key_at(lo + len) : kEmpty;
    // the team's lanes hold the keys and positions of a batch (kHeld each) and hand them around; the next batch's are on their way meanwhile
    constexpr int kHeld = kBatch > TEAM ? kBatch / TEAM : 1;
    unsigned hk[kHeld], ho[kHeld];
    const auto hold = [&](int i0) {
#pragma unroll
        for (int q = 0; q < kHeld; ++q) {
            const int i = i0 + q * TEAM + lane;
            const bool in = i < len && q * TEAM + lane < kBatch;
            const uint2 t = !in ? make_uint2(kEmpty, 0u) : FIRST ? sorted[lo + i] : make_uint2(keys[lo + i], 0u);
            hk[q] = t.x;
            ho[q] = t.y;
        }
    };
    hold(0);
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
#pragma unroll 1
    for (int i0 = 0; i0 < len; i0 += kBatch) {                       // whole teams; the shuffles stay within a team
        unsigned k[kBatch];
        nvp_vec<S, V> f[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const auto from = [&](const unsigned (&v)[kHeld]) {
                return TEAM == 64 ? (unsigned)__builtin_amdgcn_readlane((int)v[b / TEAM], b % TEAM) : (unsigned)__shfl((int)v[b / TEAM], b % TEAM, TEAM);
            };
            k[b] = from(hk);
            if (FIRST && k[b] >= (unsigned)codes) k[b] = kEmpty;
            const unsigned o = FIRST ? from(ho) : 0u;
            // first level: an entry without a row reads row 0 and drops it, so that no branch stands between the loads; later lists are mostly empty
            if (FIRST) f[b] = nvp_load_raw<S, V>(rows + (int64_t)o * dim + c);
            else if (k[b] != kEmpty && !(k[b] & kCarry)) f[b] = nvp_load_raw<S, V>(rows + (lo + i0 + b) * dim + c);
        }
        if (i0 + kBatch < len) hold(i0 + kBatch);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (k[b] == kEmpty) continue;
            const unsigned key = k[b] & ~kCarry;
            if (key != cur) {
                flush(false);
                from_left = i0 + b == 0 && same_run(before, key);
                cur = key;
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = 0.f;
            }
            if (!(k[b] & kCarry))
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += (float)f[b].v[e];
        }
    }
    flush(same_run(cur, after));
    if (next_keys && lane == 0 && blockIdx.y == 0) {
        next_keys[2 * ch] = head_key;
        next_keys[2 * ch + 1] = tail_key;
    }
}

// A list of at most kLast entries: one workgroup per entry; the entry that begins a run adds the whole run, its teams every kTeams-th entry, the teams in order.
// Most of the workgroups find no run that begins at their entry, so a workgroup is small: 256 threads (2048 entries of 1024 columns: 10.0 us, 512 threads 10.9, 1024
// 22.8 - what the launch of the waves takes).
constexpr int kLastThreads = 256;
template <typename T, int TEAM, int V>
__global__ __launch_bounds__(kLastThreads) void sum_last_kernel(const unsigned* __restrict__ keys, const float* __restrict__ rows, T* __restrict__ dtable, int m, int dim, float scale) {
    constexpr int kTeams = kLastThreads / TEAM, kBatch = 16;
    const int i = blockIdx.x;
    const unsigned key = keys[i];
    if (key == kEmpty || (key & kCarry) || (i > 0 && ((keys[i - 1] ^ key) & ~kCarry) == 0u)) return;      // a run begins with an entry that has a row
    __shared__ float part[kTeams][TEAM * V];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const bool live = (blockIdx.y * TEAM + lane) * V < dim;
    const int c = min((int)(blockIdx.y * TEAM + lane) * V, dim - V);
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    bool more = true;
    for (int e0 = i + team; more; e0 += kTeams * kBatch) {
        nvp_vec<float, V> f[kBatch];
        unsigned k[kBatch];
        bool has[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) k[b] = keys[min(e0 + b * kTeams, m - 1)];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int at = e0 + b * kTeams;
            more = at < m && k[b] != kEmpty && ((k[b] ^ key) & ~kCarry) == 0u;      // entries of a run are side by side: the last one looked at tells whether there may be more
            has[b] = more && !(k[b] & kCarry);
            f[b] = nvp_load_raw<float, V>(rows + (int64_t)(has[b] ? at : i) * dim + c);      // (no branch between the loads: an entry without a row reads the first one's)
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (has[b])
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[b].v[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) part[team][lane * V + e] = acc[e];
    __syncthreads();
    if (team == 0 && live) {
        float t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kTeams; ++k) s += part[k][lane * V + e];
            t[e] = s * scale;
        }
        nvp_store<T, V>(dtable + (int64_t)key * dim + c, t);
    }
}

// ---- few codes: sums of a chunk of rows at a time ------------------------------------------------------------------------------------------------
// With up to 1023 codes a chunk of 1024 to 8192 consecutive rows (one chunk per CU) holds every code a few times: a workgroup sorts its chunk's ids in LDS (one
// digit), adds the rows of each run up and leaves one partial row per code that is there; a second launch adds the chunks' rows in order.  dout is read once,
// chunk by chunk, so the accesses of a workgroup stay within a window of a few thousand rows (sorted over the whole batch, neighbours in the list are pages
// apart), and nothing is sorted in global memory: two launches.  Teams take equal shares of the sorted list, however the ids are distributed: a run that
// reaches into the shares behind is finished by the team it begins in, out of the sums (`head`) the others leave in LDS.
// Bound by the latency of the sort in front (11 - 14 us for few rows) and the bytes of dout behind it: 1 245 184 rows of 32 fp32 into 600 take 53 - 55 us and 6.5 for
// the second launch (159 MB and 19 MB of partial rows there and back, 3.2 TB/s; 43 us in all where dout is still in the memory-side cache).
constexpr int kLocal = 8192, kLocalWaves = 16, kLocalRounds = kLocal / (64 * kLocalWaves);      // ids of a chunk at most; a chunk has a multiple of 1024
template <typename I, typename S, int TEAM, int V>
__global__ __launch_bounds__(64 * kLocalWaves) void sum_local_kernel(const I* __restrict__ ids, const S* __restrict__ rows, float* __restrict__ part, uint8_t* __restrict__ there, int64_t n,
                                                                int chunk, int codes, int dim, int bits) {
    constexpr int kTeams = 64 * kLocalWaves / TEAM, kBatch = V > 4 ? 8 : 16, kPer = (1 << kMaxBits) / (64 * kLocalWaves);
    static_assert(kLocalWaves * (1 << kMaxBits) >= kTeams * TEAM * V, "the teams' sums take the cursors' place");
    __shared__ unsigned space[kLocalWaves << kMaxBits];                               // cursors of the waves, then the teams' first sums
    __shared__ unsigned list[kLocal];                                            // sorted: id << 16 | row of the chunk
    __shared__ unsigned wsum[kLocalWaves], length, through[kTeams];
    const int lane64 = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per_wave = chunk / kLocalWaves;
    const int64_t chunk0 = (int64_t)blockIdx.x * chunk, base = chunk0 + wave * per_wave, end = min(base + per_wave, n);
    unsigned d[kLocalRounds];
#pragma unroll
    for (int j = 0; j < kLocalRounds; ++j) d[j] = base + j * 64 + lane64 < end ? key_of(ids, base + j * 64 + lane64, codes) : 0u;
    for (int b = threadIdx.x; b < kLocalWaves << kMaxBits; b += 64 * kLocalWaves) space[b] = 0u;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kLocalRounds; ++j)
        if (base + j * 64 + lane64 < end) atomicAdd(&space[(wave << kMaxBits) + d[j]], 1u);
    __syncthreads();
    unsigned mine[kPer], sum = 0u;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int b = threadIdx.x * kPer + e;
        mine[e] = 0u;
#pragma unroll
        for (int w = 0; w < kLocalWaves; ++w) mine[e] += space[(w << kMaxBits) + b];
        sum += mine[e];
        if (b < codes) there[(int64_t)blockIdx.x * codes + b] = mine[e] ? 1 : 0;
    }
    unsigned inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(inc, o);
        if (lane64 >= o) inc += up;
    }
    if (lane64 == 63) wsum[wave] = inc;
    __syncthreads();
    unsigned here = inc - sum;
    for (int w = 0; w < wave; ++w) here += wsum[w];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int b = threadIdx.x * kPer + e;
        if (b == codes) length = here;                                           // what lies behind points nowhere
        unsigned run = here;
#pragma unroll
        for (int w = 0; w < kLocalWaves; ++w) {
            const unsigned v = space[(w << kMaxBits) + b];
            space[(w << kMaxBits) + b] = run;
            run += v;
        }
        here += mine[e];
    }
    __syncthreads();
    place_ids<kLocalRounds>(d, base, end, bits, space + (wave << kMaxBits),
                            [&](int j, unsigned at) { list[at] = d[j] << 16 | (unsigned)(wave * per_wave + j * 64 + lane64); });
    __syncthreads();

    const int len = (int)length, share = (len + kTeams - 1) / kTeams, team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const int lo = team * share, hi = min(lo + share, len);
    const bool live = lane * V < dim;
    const int c = min(lane * V, dim - V);                                        // the last vector of an odd width is moved back: its first columns are summed and written twice, alike
    float* const head = reinterpret_cast<float*>(space) + lane * V;              // [team][TEAM * V]
    float* const out = part + (int64_t)blockIdx.x * codes * dim + c;
    const S* const in = rows + chunk0 * dim + c;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    unsigned cur = 0u;
    bool to_right = false;
    if (lo < hi) {
        cur = list[lo] >> 16;
        bool from_left = lo > 0 && list[lo - 1] >> 16 == cur;                    // the run begins in a share before
        const auto flush = [&] {
            if (from_left) {
#pragma unroll
                for (int e = 0; e < V; ++e) head[team * (TEAM * V) + e] = acc[e];
            } else if (live) {
                nvp_store<float, V>(out + (int64_t)cur * dim, acc);
            }
        };
        for (int i0 = lo; i0 < hi; i0 += kBatch) {
            nvp_vec<S, V> f[kBatch];
            unsigned k[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const unsigned t = list[min(i0 + b, hi - 1)];
                k[b] = t >> 16;
                f[b] = nvp_load_raw<S, V>(in + (int64_t)(t & 0xffffu) * dim);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (i0 + b < hi) {
                    if (k[b] != cur) {
                        flush();
                        from_left = false;
                        cur = k[b];
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += (float)f[b].v[e];
                }
        }
        to_right = hi < len && list[hi] >> 16 == cur;
        if (!to_right || from_left) flush();
        if (lane == 0) through[team] = to_right && from_left;
        to_right = to_right && !from_left;                                       // the run begins here and goes on
    }
    __syncthreads();
    if (!to_right) return;
    for (int t = team + 1; t < kTeams; ++t) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += head[t * (TEAM * V) + e];
        if (!through[t]) break;
    }
    if (live) nvp_store<float, V>(out + (int64_t)cur * dim, acc);
}

// dtable[code] = scale * (the chunks' partial rows of the code, in order); a workgroup per code, its teams every kTeams-th chunk, the teams in order
template <typename T, int TEAM, int V>
__global__ __launch_bounds__(256) void sum_chunks_kernel(const float* __restrict__ part, const uint8_t* __restrict__ there, T* __restrict__ dtable, int64_t chunks, int codes, int dim, float scale) {
    constexpr int kTeams = 256 / TEAM, kBatch = V > 4 ? 8 : 16;
    __shared__ float sums[kTeams][TEAM * V];
    const int code = blockIdx.x, lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const int c = min(lane * V, dim - V);
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    for (int64_t w0 = team; w0 < chunks; w0 += kTeams * kBatch) {
        nvp_vec<float, V> f[kBatch];
        bool has[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int64_t w = min(w0 + b * kTeams, chunks - 1);
            has[b] = w0 + b * kTeams < chunks && there[w * codes + code];
            f[b] = nvp_load_raw<float, V>(part + (w * codes + code) * dim + c);  // (no branch between the loads; what is not there is dropped)
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (has[b])
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += f[b].v[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sums[team][lane * V + e] = acc[e];
    __syncthreads();
    if (team == 0 && lane * V < dim) {
        float t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float a = 0.f;
#pragma unroll
            for (int k = 0; k < kTeams; ++k) a += sums[k][lane * V + e];
            t[e] = a * scale;
        }
        nvp_store<T, V>(dtable + (int64_t)code * dim + c, t);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------
int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }
constexpr int kPerChunk2 = 32, kLast = 2560;

struct Plan {
    bool small, local;
    int passes, bits;
    int64_t radix_chunks;
    int per_chunk;                  // first level
    int levels;                     // of sum_runs_kernel
    int64_t m[12], chunks[12];      // entries (and, behind them, those of the list that is left) and chunks of each level
    int64_t last;                   // entries for sum_last_kernel, 0: nothing left
    int64_t off_sorted[2], off_count, off_total, off_lkey[2], off_lrow[2], bytes;
};
Plan plan_of(int64_t n, int64_t codes, int64_t dim) {
    Plan P{};
    // chunk by chunk or sorted as a whole, us of kernels, fp32: 600 codes x 32: 64 rows 11 / 12.5, 4096 rows 14 / 22, 65 536 rows 16 / 32, 1 245 184 rows 43 / 67;
    // x 64: 1 245 184 rows 90 / 106;  x 114: 65 536 rows 27 / 36, 262 144 rows 51 / 54, 1 245 184 rows 177 / 165;  1000 codes x 256: 16 384 rows 39 / 26, 262 144 rows
    // 138 / 71 (few teams of many lanes, and a fourth of a chunk's bytes again in partial rows)
    P.local = n && codes < (1 << kMaxBits) && (dim <= 64 || (dim <= 128 && n <= 1 << 18));
    if (P.local) {
        // a chunk per CU, as long as its ids fit; equal chunks where there are more
        const int64_t rounds = (n + 256 * kLocal - 1) / (256 * kLocal);
        P.per_chunk = (int)((n + 256 * rounds * 1024 - 1) / (256 * rounds * 1024)) * 1024;
        P.chunks[0] = (n + P.per_chunk - 1) / P.per_chunk;
        for (P.bits = 1; (codes >> P.bits) != 0;) ++P.bits;                      // keys 0 .. codes
        P.off_total = up256(P.chunks[0] * codes * dim * 4);
        P.bytes = P.off_total + up256(P.chunks[0] * codes);
        return P;
    }
    P.small = n <= kSmall;
    int b = 1;
    while (b < 32 && ((codes + 1) - 1) >> b) ++b;                    // keys 0 .. codes
    P.passes = (b + kMaxBits - 1) / kMaxBits;
    P.bits = (b + P.passes - 1) / P.passes;
    P.radix_chunks = (n + kChunk - 1) / kChunk;
    // entries per team at the first level: enough teams to keep the chip's memory busy (256 CUs x 8 waves), and no fewer entries than that allows, because every
    // chunk may leave two partial rows behind
    const int64_t waves = n * ((dim * 4 + 1023) / 1024) * (dim >= 256 ? 64 : dim >= 128 ? 32 : dim >= 64 ? 16 : 8) / 64;
    P.per_chunk = 16;
    while (P.per_chunk < 128 && waves / (2 * P.per_chunk) >= 2048) P.per_chunk *= 2;
    int64_t m = n;
    for (P.levels = 0, P.last = 0;;) {
        P.m[P.levels] = m;
        P.chunks[P.levels] = (m + (P.levels ? kPerChunk2 : P.per_chunk) - 1) / (P.levels ? kPerChunk2 : P.per_chunk);
        m = P.chunks[P.levels] <= 1 ? 0 : 2 * P.chunks[P.levels];
        P.m[++P.levels] = m;
        if (m <= kLast) break;
    }
    P.last = m;
    int64_t at = 0;
    for (int i = 0; i < (P.small ? 1 : 2); ++i) {
        P.off_sorted[i] = at;
        at += up256(n * 8);
    }
    P.off_count = at;
    if (!P.small) at += up256(P.radix_chunks * (1ll << P.bits) * 4);
    P.off_total = at;
    if (!P.small) at += up256((1ll << P.bits) * 4);
    for (int i = 0; i < 2; ++i) {                                    // level l writes list l & 1: a later list is never longer than the one it replaces
        const int64_t e = i + 1 <= P.levels ? P.m[i + 1] : 0;
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

// calls `f` with the team's size as a constant
template <typename F> void with_team(int team, F f) {
    if (team == 4) f(std::integral_constant<int, 4>());
    else if (team == 8) f(std::integral_constant<int, 8>());
    else if (team == 16) f(std::integral_constant<int, 16>());
    else if (team == 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}

constexpr int64_t kMaxGroups = ((1ll << 32) - 1) / 256;                                     // workgroups of 256 threads: a launch has fewer than 2^32 threads along x
template <typename T, typename O, typename I, int V>
int fwd(const I* ids, const T* table, O* out, int64_t n, int64_t codes, int dim, float scale, hipStream_t st) {
    const int team = team_of((dim + V - 1) / V);
    const int64_t per = 4 * (256 / team), most = kMaxGroups * per;                            // rows of a workgroup, of a launch
    for (int64_t r = 0; r < n; r += most) {
        const int64_t here = n - r < most ? n - r : most;
        const dim3 g((unsigned)((here + per - 1) / per)), wg(256);
        with_team(team, [&](auto t) { hipLaunchKernelGGL((lookup_fwd_kernel<T, O, I, decltype(t)::value, V>), g, wg, 0, st, ids + r, table, out + r * dim, here, codes, dim, scale); });
        NVP_LAUNCH_CHECK();
    }
    return 0;
}

template <typename S, typename T, bool FIRST, int V>
int sum_level(const uint2* sorted, const unsigned* keys, const S* rows, T* dtable, unsigned* nkeys, float* nrows, int64_t m, int per_chunk, int64_t chunks, int64_t codes, int dim, float scale,
              bool filled, hipStream_t st) {
    const int team = team_of((dim + V - 1) / V), teams = 256 / team;
    const int64_t sums = (chunks + teams - 1) / teams, fill = FIRST && !filled ? (codes + 255) / 256 : 0, cols = (dim + team * V - 1) / (team * V);
    if (sums + fill > kMaxGroups || cols > 65535) return NVP_ERR_UNSUPPORTED;
    with_team(team, [&](auto t) {
        hipLaunchKernelGGL((sum_runs_kernel<S, T, FIRST, decltype(t)::value, V>), dim3((unsigned)(sums + fill), (unsigned)cols), dim3(256), 0, st, sorted, keys, rows, dtable, nkeys, nrows, m,
                           per_chunk, chunks, sums, codes, dim, scale);
    });
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename S, typename T, int V, int VF>
int sums(const Plan& P, const uint2* sorted, const S* dout, T* dtable, uint8_t* ws, int64_t codes, int dim, float scale, bool filled, hipStream_t st) {
    const auto lkey = [&](int l) { return (unsigned*)(ws + P.off_lkey[l & 1]); };
    const auto lrow = [&](int l) { return (float*)(ws + P.off_lrow[l & 1]); };
    int rc = 0;
    for (int l = 0; !rc && l < P.levels; ++l) {
        unsigned* nk = P.m[l + 1] ? lkey(l) : nullptr;
        float* nr = P.m[l + 1] ? lrow(l) : nullptr;
        rc = l == 0 ? sum_level<S, T, true, V>(sorted, nullptr, dout, dtable, nk, nr, P.m[0], P.per_chunk, P.chunks[0], codes, dim, scale, filled, st)
                    : sum_level<float, T, false, VF>(nullptr, lkey(l - 1), lrow(l - 1), dtable, nk, nr, P.m[l], kPerChunk2, P.chunks[l], codes, dim, scale, filled, st);
    }
    if (rc || !P.last) return rc;
    const int team = team_of((dim + VF - 1) / VF);
    with_team(team, [&](auto t) {
        hipLaunchKernelGGL((sum_last_kernel<T, decltype(t)::value, VF>), dim3((unsigned)P.last, (unsigned)((dim + team * VF - 1) / (team * VF))), dim3(kLastThreads), 0, st, lkey(P.levels - 1),
                           lrow(P.levels - 1), dtable, (int)P.last, dim, scale);
    });
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename I, typename S, typename T, int V>
int sums_local(const Plan& P, const I* ids, const S* dout, T* dtable, uint8_t* ws, int64_t n, int64_t codes, int dim, float scale, hipStream_t st) {
    float* const part = (float*)ws;
    uint8_t* const there = ws + P.off_total;
    const int team = team_of((dim + V - 1) / V);
    if (P.chunks[0] > kMaxGroups / 4) return NVP_ERR_UNSUPPORTED;
    with_team(team, [&](auto t) {
        hipLaunchKernelGGL((sum_local_kernel<I, S, decltype(t)::value, V>), dim3((unsigned)P.chunks[0]), dim3(64 * kLocalWaves), 0, st, ids, dout, part, there, n, P.per_chunk, (int)codes, dim, P.bits);
    });
    NVP_LAUNCH_CHECK();
    with_team(team, [&](auto t) {
        hipLaunchKernelGGL((sum_chunks_kernel<T, decltype(t)::value, V>), dim3((unsigned)codes), dim3(256), 0, st, part, there, dtable, P.chunks[0], (int)codes, dim, scale);
    });
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename I, typename S, typename T>
int bwd(const I* ids, const S* dout, T* dtable, int64_t n, int64_t codes, int dim, float scale, uint8_t* ws, hipStream_t st) {
    const Plan P = plan_of(n, codes, dim);
    constexpr int VL = 16 / sizeof(S);
    if (P.local) return dim >= VL ? sums_local<I, S, T, VL>(P, ids, dout, dtable, ws, n, codes, dim, scale, st) : sums_local<I, S, T, 1>(P, ids, dout, dtable, ws, n, codes, dim, scale, st);
    uint2* buf[2] = {(uint2*)(ws + P.off_sorted[0]), (uint2*)(ws + P.off_sorted[P.small ? 0 : 1])};
    // zeros first, beside the sort, where three quarters of the rows stay empty (the others are written twice): us, fp32, zeros behind the sort / beside it,
    // 65 536 codes x 1024: 512 ids 48 / 40, 16 384 ids 110 / 99;  65 536 codes x 512: 32 768 ids 59 / 63, 65 536 ids 80 / 85
    const int64_t bytes = codes * (int64_t)dim * (int64_t)sizeof(T), launches = P.small ? 1 : 3 * P.passes;
    const int64_t slice = ((bytes + launches - 1) / launches + kFillBytes - 1) / kFillBytes * kFillBytes;
    const bool filled = n && codes >= 4 * n && slice / kFillBytes < (1 << 21);      // (workgroups of up to 1024 threads)
    int64_t done = 0;
    const auto next = [&](int64_t work, int64_t& grid) {                         // the launch's grid with its part of the table
        const int64_t len = filled ? (bytes - done < slice ? bytes - done : slice) : 0;
        const Fill f{(uint8_t*)dtable + done, len, (unsigned)work};
        done += len;
        grid = work + (len + kFillBytes - 1) / kFillBytes;
        return f;
    };
    int at = 0;
    int64_t g;
    if (n == 0) {
        // nothing to sort: the sums below only write zeros
    } else if (P.small) {
        int padded = 2;
        while (padded < n) padded <<= 1;
        const Fill f = next(1, g);
        hipLaunchKernelGGL((sort_small_kernel<I>), dim3((unsigned)g), dim3(1024), 0, st, ids, buf[0], (int)n, codes, padded, f);
        NVP_LAUNCH_CHECK();
    } else {
        unsigned *count = (unsigned*)(ws + P.off_count), *total = (unsigned*)(ws + P.off_total);
        const dim3 wg(256), wide(64 * kWaves);
        for (int p = 0; p < P.passes; ++p) {
            const int shift = p * P.bits;
            Fill f = next(P.radix_chunks, g);
            if (p == 0) hipLaunchKernelGGL((radix_count_kernel<I, true>), dim3((unsigned)g), wg, 0, st, ids, buf[at], count, n, codes, shift, P.bits, f);
            else hipLaunchKernelGGL((radix_count_kernel<I, false>), dim3((unsigned)g), wg, 0, st, ids, buf[at], count, n, codes, shift, P.bits, f);
            NVP_LAUNCH_CHECK();
            f = next(((1 << P.bits) + 15) / 16, g);
            hipLaunchKernelGGL(radix_scan_kernel, dim3((unsigned)g), dim3(1024), 0, st, count, total, (int)P.radix_chunks, P.bits, f);
            NVP_LAUNCH_CHECK();
            f = next(P.radix_chunks, g);
            if (p == 0) hipLaunchKernelGGL((radix_scatter_kernel<I, true>), dim3((unsigned)g), wide, 0, st, ids, buf[at], count, total, buf[at ^ 1], n, codes, shift, P.bits, f);
            else hipLaunchKernelGGL((radix_scatter_kernel<I, false>), dim3((unsigned)g), wide, 0, st, ids, buf[at], count, total, buf[at ^ 1], n, codes, shift, P.bits, f);
            NVP_LAUNCH_CHECK();
            at ^= 1;
        }
    }
    constexpr int V = vec_of<S, T>();
    if (dim >= (V > 4 ? V : 4)) return sums<S, T, V, 4>(P, buf[at], dout, dtable, ws, codes, dim, scale, filled, st);
    return sums<S, T, 1, 1>(P, buf[at], dout, dtable, ws, codes, dim, scale, filled, st);
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
