// Drawing one token a row from logits l [B, V], given a random number u from [0, 1) for each row:
//
//   w_i = e^((l_i - max l) / T)                            weights in 64 bits; -inf and NaN have none
//   order: descending l, the lowest index of equal ones first
//   top_k: the first k of it stay; top_p: of those the shortest run that holds p of their weight at least; min_p: of those what has w >= min_p
//   the token: the first in the order of the vocabulary up to which the weights that stay come to more than u of their sum
//
// What stays is a run of the order whatever the filters are, so it is held as its last element: a key (the bits of l, made to order like l) and, among equal keys, an index.
// A row is cut into segments of 1024 neighbours, one wavefront's 16 values a lane, whose maxima and sums are what the draw goes by: it finds its segment, then its token in it.
//
// Three kernels.  One workgroup for each slice of 16 segments reads the logits: segments' maxima; without filters their sums too; with top_k or top_p a histogram of the slice, counts and weights by
// l / T in steps of 1 / 16, on one grid for the row.  With filters the slices' workgroups add up the row's histograms, which shows the bin in which the run ends, and collect what lies in it and above, or,
// where that is more than a list holds, what lies in it and the sums of what lies above.  One workgroup a row finishes: it sorts the list, which settles the run, and draws.
// Rows that this does not suit (more than a list of equal or nearly equal logits in the last bin, 2^50 bins and more) are worked on by that one workgroup alone, a pass over the row for every eight bits of the key.
#include "sample.hpp"

#include "ffn.hpp"

namespace mmx {

constexpr int SEG = 1024, SLICE = 16;     // logits of a segment, segments of a slice
constexpr int BINS = 512;                 // the last one: everything below
constexpr double PER_UNIT = 16;           // bins of a unit of l / T
constexpr int LIST = 4096;                // entries
constexpr int MOST_SUMS = 1024;           // segments of a row whose sums fit beside a list
constexpr double GRID = 1125899906842624.0;  // 2^50: up to here bins are exact
constexpr float NEVER = -__builtin_huge_valf();

// What a row asks for
struct RowAsks {
    double T, p, min_p;
    int k;
    bool greedy, top_k, top_p, min;
    __device__ __forceinline__ bool filtered() const { return !greedy && (top_k || top_p); }
};
__device__ __forceinline__ RowAsks asks_of(const SampleArgs& a, int row) {
    RowAsks r;
    r.T = a.temperature ? (double)a.temperature[row] : a.temperature_all;
    r.k = a.top_k ? a.top_k[row] : a.top_k_all;
    r.p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
    r.min_p = a.min_p ? (double)a.min_p[row] : a.min_p_all;
    r.top_k = r.k > 0 && r.k < a.V;
    r.top_p = r.p < 1.0;
    r.min = r.min_p > 0.0;
    r.greedy = !(r.T > 0.0) || r.k == 1 || r.p <= 0.0;
    return r;
}

// Orders like the value; the two zeros are one (values come through `settled`).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = f2u(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return u2f(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float settled(float x) { return x != x ? NEVER : x + 0.0f; }

__device__ __forceinline__ double weight_of(float l, float top, double T) {
    if (l == top) return 1.0;  // (an infinite one too: the others have no weight beside it)
    return l == NEVER ? 0.0 : exp(((double)l - (double)top) / T);
}

__device__ __forceinline__ float value_at(const uint16_t* row, int64_t i) { return settled(from_bf16(row[i])); }
__device__ __forceinline__ float value_at(const float* row, int64_t i) { return settled(row[i]); }

// The 16 values of a lane in a segment and where in the segment they lie: pieces of 16 bytes, a wavefront's one behind the other.
template <typename TL>
struct Lane16 {
    static constexpr int PER = 16 / (int)sizeof(TL);  // values of a piece
    float v[16];
    __device__ __forceinline__ static int at(int e) { return (e / PER) * (64 * PER) + (threadIdx.x & 63) * PER + e % PER; }
    __device__ __forceinline__ void load(const TL* row, int V, int seg) {
        const int64_t base = (int64_t)seg * SEG;
        if (base + SEG <= V) {
            u32x4 w[16 / PER];
#pragma unroll
            for (int c = 0; c < 16 / PER; c++) __builtin_memcpy(&w[c], __builtin_assume_aligned(row + base + at(c * PER), sizeof(TL)), 16);  // (the hardware takes any address)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t x = w[e / PER][(e % PER) * (int)sizeof(TL) / 4];
                if constexpr (sizeof(TL) == 2) v[e] = settled(u2f(e & 1 ? x & 0xffff0000u : x << 16));
                else v[e] = settled(u2f(x));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = base + at(e) < V ? value_at(row, base + at(e)) : NEVER;
        }
    }
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

constexpr int NW = 16, THREADS = NW * 64;

struct Cut {       // what stays: keys above, and of the equal ones indexes up to `index`
    uint32_t key;
    int index;
    __device__ __forceinline__ bool holds(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

// What a slice's workgroup leaves
struct Slice {
    double bin;  // of its largest logit
    unsigned long long mass;
    float top;
    uint32_t count;
};
enum { BY_LIST, BY_SUMS, ALONE };
struct State {
    uint32_t entries, path, before_count;
    float top;
    double before_mass, mass;  // of what lies above the last bin, and of everything
};
// A row's scratch
struct Scratch {
    float* seg_top;
    double* sums;
    Slice* slices;
    State* state;
    unsigned long long* list;
    unsigned long long* mass;  // histograms, a slice's behind the other
    uint32_t* count;
    int segs, n_slices;
};
__host__ __device__ inline size_t row_bytes(int V) {
    const size_t segs = ((size_t)V + SEG - 1) / SEG, slices = (segs + SLICE - 1) / SLICE;
    return (segs * 12 + slices * (sizeof(Slice) + BINS * 12) + LIST * 8 + sizeof(State) + 255) & ~(size_t)255;
}
__device__ __forceinline__ Scratch scratch_of(const SampleArgs& a, int row) {
    Scratch r;
    r.segs = (a.V + SEG - 1) / SEG;
    r.n_slices = (r.segs + SLICE - 1) / SLICE;
    char* p = a.scratch + (int64_t)row * row_bytes(a.V);
    r.list = reinterpret_cast<unsigned long long*>(p), p += LIST * 8;
    r.state = reinterpret_cast<State*>(p), p += sizeof(State);
    r.slices = reinterpret_cast<Slice*>(p), p += r.n_slices * sizeof(Slice);
    r.mass = reinterpret_cast<unsigned long long*>(p), p += (int64_t)r.n_slices * BINS * 8;
    r.sums = reinterpret_cast<double*>(p), p += (int64_t)r.segs * 8;
    r.seg_top = reinterpret_cast<float*>(p), p += (int64_t)r.segs * 4;
    r.count = reinterpret_cast<uint32_t*>(p);
    return r;
}
static_assert(sizeof(Slice) % 8 == 0 && sizeof(State) % 8 == 0, "what lies behind them stays aligned");

__device__ __forceinline__ unsigned long long whole(double w, double scale) { return (unsigned long long)(w * scale + 0.5); }

struct Shared {
    unsigned long long mass[256];
    uint32_t count[256];
    double part[NW];
    float fpart[NW];
    uint32_t bin, found;
    unsigned long long before_mass;
    uint32_t before_count;
    int pick;
    double rest;
};

// A value of each thread: the sum over the threads before it, and over all
__device__ __forceinline__ double scan_before(double v, double* part, double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double run = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(run, d);
        if (lane >= d) run += o;
    }
    __syncthreads();
    if (lane == 63) part[wave] = run;
    __syncthreads();
    double before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        before += w < wave ? part[w] : 0.0;
        total += part[w];
    }
    *all = total;
    return before + run - v;
}

// The cut that keeps the first `want_count` of what `limit` holds (by_mass: the shortest run of it that holds `want_mass`): its key by eight bits at a time from the top, over the whole row each time,
// then, if not all of the equal keys stay, the index.  Masses are whole numbers of 2^-shift, whose sums do not depend on their order.
template <typename TL>
__device__ Cut select(const TL* row, int V, float top, double T, double scale, Cut limit, bool by_mass, uint32_t want_count, unsigned long long want_mass, Shared& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, segs = (V + SEG - 1) / SEG;
    uint32_t prefix = 0;
    unsigned long long mass_before = 0;
    uint32_t count_before = 0, equal = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += THREADS) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        for (int g = wave; g < segs; g += NW) {
            Lane16<TL> x;
            x.load(row, V, g);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t k = key_of(x.v[e]);
                if (x.v[e] == NEVER || !limit.holds(k, g * SEG + x.at(e)) || (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
                atomicAdd(&s.count[k >> shift & 255], 1u);
                if (by_mass) atomicAdd(&s.mass[k >> shift & 255], whole(weight_of(x.v[e], top, T), scale));
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t c = count_before, last = 0;
            unsigned long long m = mass_before, last_m = m;
            uint32_t last_c = c;
            for (int b = 255; b >= 0; b--) {
                if (!s.count[b]) continue;
                last = b, last_c = c, last_m = m;
                c += s.count[b];
                m += s.mass[b];
                if (by_mass ? m >= want_mass : c >= want_count) break;
            }
            s.bin = last, s.before_count = last_c, s.before_mass = last_m;
        }
        __syncthreads();
        prefix |= s.bin << shift;
        count_before = s.before_count, mass_before = s.before_mass, equal = s.count[s.bin];
    }
    uint32_t stay = want_count - count_before;
    if (by_mass) {
        const unsigned long long each = whole(weight_of(of_key(prefix), top, T), scale);
        const unsigned long long n = each ? (want_mass - mass_before + each - 1) / each : equal;
        stay = want_mass <= mass_before ? 1 : n < equal ? (uint32_t)n : equal;
    }
    if (stay >= equal) return Cut{prefix, prefix == limit.key ? limit.index : V};
    // the index of equal key number `stay`
    uint32_t seen = 0;
    Cut cut = {prefix, V};
    for (int g0 = 0; g0 < segs; g0 += NW) {
        const int g = g0 + wave;
        uint32_t n = 0;
        Lane16<TL> x;
        if (g < segs) {
            x.load(row, V, g);
#pragma unroll
            for (int e = 0; e < 16; e++) n += key_of(x.v[e]) == prefix && limit.holds(prefix, g * SEG + x.at(e));
        }
        const uint32_t all = wave_sum(n);
        __syncthreads();
        if (lane == 0) s.count[wave] = all;
        __syncthreads();
        for (int w = 0; w < NW; w++) {
            if (seen + s.count[w] >= stay) {  // (the same in all threads)
                const int seg = g0 + w;
                if (threadIdx.x == 0) {
                    uint32_t left = stay - seen;
                    for (int i = seg * SEG; i < V; i++)
                        if (key_of(value_at(row, i)) == prefix && --left == 0) {
                            s.pick = i;
                            break;
                        }
                }
                __syncthreads();
                cut.index = s.pick;
                return cut;
            }
            seen += s.count[w];
        }
    }
    return cut;
}

// ---- the slices -----------------------------------------------------------------------------------------------------------------
template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_slices_kernel(const SampleArgs a) {
    __shared__ unsigned long long mass[BINS], total_mass;
    __shared__ uint32_t count[BINS], total_count;
    __shared__ float tops[NW];
    const int row_at = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Scratch sc = scratch_of(a, row_at);
    const RowAsks r = asks_of(a, row_at);
    const int g = blockIdx.x * SLICE + wave;
    const bool here = g < sc.segs;
    Lane16<TL> x;
    float top = NEVER;
    if (here) {
        x.load(reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld), a.V, g);
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, x.v[e]);
        top = wave_max(top);
        if (lane == 0) sc.seg_top[g] = top;
    }
    if (!r.filtered()) {
        if (!here || r.greedy || r.min) return;
        double w = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) w += weight_of(x.v[e], top, r.T);
        w = wave_sum(top == NEVER ? 0.0 : w);
        if (lane == 0) sc.sums[g] = w;
        return;
    }
    if (lane == 0) tops[wave] = top;
    for (int i = threadIdx.x; i < BINS; i += THREADS) mass[i] = 0, count[i] = 0;
    if (threadIdx.x == 0) total_mass = 0, total_count = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, tops[w]);
    const double per = PER_UNIT / r.T, bin = floor((double)top * per), scale = (double)(1ull << a.shift);
    if (top != NEVER && here) {
        unsigned long long m = 0;
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (x.v[e] == NEVER) continue;
            const double d = bin - floor((double)x.v[e] * per);
            const int at = d < BINS - 1 ? (int)d : BINS - 1;
            const unsigned long long w = whole(weight_of(x.v[e], top, r.T), scale);
            atomicAdd(&count[at], 1u);
            atomicAdd(&mass[at], w);
            m += w, n++;
        }
        m = wave_sum(m), n = wave_sum(n);
        if (lane == 0) atomicAdd(&total_mass, m), atomicAdd(&total_count, n);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS) {
        sc.mass[(int64_t)blockIdx.x * BINS + i] = mass[i];
        sc.count[(int64_t)blockIdx.x * BINS + i] = count[i];
    }
    if (threadIdx.x == 0) {
        sc.slices[blockIdx.x] = Slice{bin, total_mass, top, total_count};
        if (blockIdx.x == 0) sc.state->entries = 0;
    }
}

// ---- what the filters leave -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float row_top(const Scratch& sc, float* part) {
    float top = NEVER;
    for (int i = threadIdx.x; i < sc.segs; i += THREADS) top = fmaxf(top, sc.seg_top[i]);
    top = wave_max(top);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, part[w]);
    return top;
}

template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_filter_kernel(const SampleArgs a) {
    __shared__ double part[NW];
    __shared__ float fpart[NW];
    __shared__ uint32_t found, entries, base, n_last, n_run;
    __shared__ double before_mass, before_count;
    const int row_at = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Scratch sc = scratch_of(a, row_at);
    const RowAsks r = asks_of(a, row_at);
    if (r.greedy || !(r.filtered() || r.min)) return;
    const float top = row_top(sc, fpart);
    if (top == NEVER) return;
    const int g = blockIdx.x * SLICE + wave;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    const bool here = g < sc.segs;
    const float seg_top = here ? sc.seg_top[g] : NEVER;
    if (!r.filtered()) {
        if (!here) return;
        double w = 0;
        if (seg_top != NEVER) {
            Lane16<TL> x;
            x.load(row, a.V, g);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const double v = weight_of(x.v[e], top, r.T);
                w += v < r.min_p && x.v[e] != top ? 0.0 : v;
            }
            w = wave_sum(w);
        }
        if (lane == 0) sc.sums[g] = w;
        return;
    }
    // the row's histogram, a bin a thread
    double bin = -__builtin_huge_val(), all_mass = 0, all_count = 0;
    for (int i = 0; i < sc.n_slices; i++) {
        const Slice s = sc.slices[i];
        if (s.count) bin = fmax(bin, s.bin);
    }
    const double per = PER_UNIT / r.T;
    const bool odd = !(fabs(bin) <= GRID) || !(per <= 1e300);  // (a slice that lies below the grid has all it holds in the last bin)
    const double scale = 1.0 / (double)(1ull << a.shift);
    const int b = threadIdx.x;
    double mass = 0, count = 0;
    if (!odd) {
        for (int i = 0; i < sc.n_slices; i++) {
            const Slice s = sc.slices[i];
            if (!s.count) continue;
            const double f = weight_of(s.top, top, r.T) * scale;
            all_mass += f * (double)s.mass, all_count += s.count;
            const double at = b - (bin - s.bin);
            if (b < BINS - 1 && at >= 0.0) {
                const int64_t o = (int64_t)i * BINS + (int)at;
                mass += f * (double)sc.mass[o];
                count += sc.count[o];
            }
        }
    }
    double sum_mass, sum_count;
    double run_mass = scan_before(mass, part, &sum_mass), run_count = scan_before(count, part, &sum_count);
    if (b == BINS - 1) mass = fmax(all_mass - sum_mass, 0.0), count = all_count - sum_count;
    // the bin in which the run ends: of top_k the first whose count is enough, of top_p alone the first whose mass is (of both: top_p's share is of what top_k leaves, which only the list tells)
    __syncthreads();
    if (threadIdx.x == 0) found = BINS - 1;
    __syncthreads();
    if (b < BINS && (r.top_k ? run_count + count >= (double)r.k : run_mass + mass >= r.p * all_mass)) atomicMin(&found, (uint32_t)b);
    __syncthreads();
    const int cut = found;
    if (b == cut) before_mass = run_mass, before_count = run_count, n_last = (uint32_t)count, n_run = (uint32_t)(run_count + count);
    if (threadIdx.x == 0) entries = 0;
    __syncthreads();
    const uint32_t path = odd ? ALONE : n_run <= LIST ? BY_LIST : (r.top_k && r.top_p) || n_last > LIST || sc.segs > MOST_SUMS ? ALONE : BY_SUMS;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        State* const s = sc.state;
        s->path = path, s->before_count = (uint32_t)before_count, s->top = top, s->before_mass = before_mass, s->mass = all_mass;
    }
    if (path == ALONE) return;
    // this slice's: into the list what lies in the bin (BY_LIST: and above it), into the sums what lies above
    Lane16<TL> x;
    uint32_t takes = 0;
    const bool some = here && seg_top != NEVER && bin - floor((double)seg_top * per) <= cut;
    double w = 0;
    if (some) {
        x.load(row, a.V, g);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (x.v[e] == NEVER) continue;
            const double d = fmin(bin - floor((double)x.v[e] * per), BINS - 1.0);
            if (d == cut || (path == BY_LIST && d < cut)) takes |= 1u << e;
            if (path == BY_SUMS && d < cut) {
                const double v = weight_of(x.v[e], top, r.T);
                w += v < r.min_p && x.v[e] != top ? 0.0 : v;
            }
        }
    }
    if (path == BY_SUMS && here) {
        w = wave_sum(w);
        if (lane == 0) sc.sums[g] = w;
    }
    uint32_t at = 0;
    if (takes) at = atomicAdd(&entries, (uint32_t)__popc(takes));
    __syncthreads();
    if (threadIdx.x == 0 && entries) base = atomicAdd(&sc.state->entries, entries);
    __syncthreads();
    if (takes) {
        at += base;
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (takes >> e & 1) sc.list[at++] = (unsigned long long)key_of(x.v[e]) << 32 | (0xffffffffu - (uint32_t)(g * SEG + x.at(e)));
    }
}

// ---- the draw: a workgroup a row -------------------------------------------------------------------------------------------------
// n entries of the list, largest first; returns the place of them
__device__ unsigned long long* sorted(unsigned long long* e, unsigned long long* room, int n) {
    if (n <= THREADS) {  // by counting
        const unsigned long long mine = (int)threadIdx.x < n ? e[threadIdx.x] : 0;
        int rank = 0;
        if ((int)threadIdx.x < n)
            for (int i = 0; i < n; i++) rank += e[i] > mine;
        if ((int)threadIdx.x < n) room[rank] = mine;
        __syncthreads();
        return room;
    }
    int m = 2048;
    while (m < n) m *= 2;
    for (int i = n + threadIdx.x; i < m; i += THREADS) e[i] = 0;
    for (int k = 2; k <= m; k *= 2)
        for (int d = k / 2; d >= 1; d /= 2) {
            __syncthreads();
            for (int t = threadIdx.x; t < m / 2; t += THREADS) {
                const int i = (t / d) * 2 * d + t % d;
                const unsigned long long p = e[i], q = e[i + d];
                if ((p < q) == ((i & k) == 0)) e[i] = q, e[i + d] = p;
            }
        }
    __syncthreads();
    return e;
}

template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_draw_kernel(const SampleArgs a) {
    __shared__ Shared s;
    __shared__ unsigned long long list[LIST], room[THREADS];
    const int row_at = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int V = a.V;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    const Scratch sc = scratch_of(a, row_at);
    const int segs = sc.segs;
    const RowAsks r = asks_of(a, row_at);
    const float top = row_top(sc, s.fpart);
    if (top == NEVER) {
        if (threadIdx.x == 0) a.ids[row_at] = -1;
        return;
    }
    const double u = (double)a.u[row_at];
    if (r.greedy) {  // the first segment that holds it, its first place in it
        if (threadIdx.x == 0) s.pick = V;
        __syncthreads();
        for (int g = threadIdx.x; g < segs; g += THREADS)
            if (sc.seg_top[g] == top) atomicMin(&s.pick, g);
        __syncthreads();
        const int i = s.pick * SEG + threadIdx.x;
        if (threadIdx.x == 0) s.found = 0xffffffffu;
        __syncthreads();
        if (i < V && value_at(row, i) == top) atomicMin(&s.found, (uint32_t)i);
        __syncthreads();
        if (threadIdx.x == 0) a.ids[row_at] = (int)s.found;
        return;
    }
    const uint32_t path = r.filtered() ? sc.state->path : BY_SUMS;
    const double scale = (double)(1ull << a.shift);
    Cut cut = {key_of(NEVER), V};
    double* const sums = sc.sums;
    auto stays = [&](float l, int i) __attribute__((always_inline)) {
        if (l == NEVER || !cut.holds(key_of(l), i)) return 0.0;
        const double w = weight_of(l, top, r.T);
        return w < r.min_p && l != top ? 0.0 : w;
    };
    if (r.filtered() && path != ALONE) {
        const int n = (int)sc.state->entries;
        for (int i = threadIdx.x; i < n; i += THREADS) list[i] = sc.list[i];
        __syncthreads();
        unsigned long long* const e = sorted(list, room, n);
        // how many of the list stay: four neighbours a thread, their weights and the weight in front of them
        double w[LIST / THREADS], mine = 0, total;
        const int i0 = threadIdx.x * (LIST / THREADS);
#pragma unroll
        for (int c = 0; c < LIST / THREADS; c++) {
            const int i = i0 + c;
            // (above the bin are, by sums, before_count more)
            const bool in = i < n && (!r.top_k || i + (path == BY_SUMS ? (int)sc.state->before_count : 0) < r.k);
            w[c] = in ? weight_of(of_key((uint32_t)(e[i] >> 32)), top, r.T) : -1.0;
            mine += in ? w[c] : 0.0;
        }
        double before = scan_before(mine, s.part, &total);
        if (path == BY_SUMS) before += sc.state->before_mass;
        const double want = r.p * (r.top_k ? total : sc.state->mass);
        uint32_t kept = 0;
#pragma unroll
        for (int c = 0; c < LIST / THREADS; c++) {
            // (of a run by mass the one that reaches it is the last; one token at least)
            const bool in = w[c] >= 0.0 && (!r.top_p || before < want || i0 + c == 0);
            if (w[c] >= 0.0) before += w[c];
            if (in) kept = i0 + c + 1;
        }
        if (threadIdx.x == 0) s.found = 0;
        __syncthreads();
        atomicMax(&s.found, kept);
        __syncthreads();
        kept = s.found;
        const unsigned long long last = e[kept - 1];
        cut = Cut{(uint32_t)(last >> 32), (int)(0xffffffffu - (uint32_t)last)};
        if (path == BY_LIST) {
            // in the order of the vocabulary: the same once more by index (the order is that of falling complements)
            __syncthreads();
            for (int i = threadIdx.x; i < (int)kept; i += THREADS) e[i] = e[i] << 32 | e[i] >> 32;
            __syncthreads();
            unsigned long long* const o = sorted(e, e == list ? room : list, (int)kept);
            double run = 0;
#pragma unroll
            for (int c = 0; c < LIST / THREADS; c++) {
                const int i = i0 + c;
                w[c] = i < (int)kept ? stays(of_key((uint32_t)o[i]), -1) : 0.0;
                run += w[c];
            }
            double all, at = scan_before(run, s.part, &all);
            const double goal = u > 0.0 ? u * all : 0.0;
            if (threadIdx.x == 0) s.found = 0xffffffffu, s.bin = 0;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < LIST / THREADS; c++) {
                if (w[c] <= 0.0) continue;
                at += w[c];
                if (at > goal) atomicMin(&s.found, (uint32_t)(i0 + c));
                atomicMax(&s.bin, (uint32_t)(i0 + c));
            }
            __syncthreads();
            if (threadIdx.x == 0) a.ids[row_at] = (int)(0xffffffffu - (uint32_t)(o[s.found != 0xffffffffu ? s.found : s.bin] >> 32));
            return;
        }
        // what stays of the bin, to its segments' sums
        unsigned long long* const more = e == list ? room : list;
        for (int g = threadIdx.x; g < segs; g += THREADS) more[g] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < (int)kept; i += THREADS) {
            const double v = weight_of(of_key((uint32_t)(e[i] >> 32)), top, r.T);
            if (!(v < r.min_p)) atomicAdd(&more[(0xffffffffu - (uint32_t)e[i]) / SEG], whole(v, scale));
        }
        __syncthreads();
        for (int g = threadIdx.x; g < segs; g += THREADS) sums[g] += (double)more[g] / scale;
    } else if (path == ALONE) {
        if (r.top_k) cut = select(row, V, top, r.T, scale, cut, false, (uint32_t)r.k, 0ull, s);
        if (r.top_p) {
            unsigned long long m = 0;
            for (int g = wave; g < segs; g += NW) {
                Lane16<TL> x;
                x.load(row, V, g);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (cut.holds(key_of(x.v[e]), g * SEG + x.at(e))) m += whole(weight_of(x.v[e], top, r.T), scale);
            }
            m = wave_sum(m);
            __syncthreads();
            if (lane == 0) s.mass[wave] = m;
            __syncthreads();
            m = 0;
            for (int w = 0; w < NW; w++) m += s.mass[w];
            cut = select(row, V, top, r.T, scale, cut, true, 0u, (unsigned long long)ceil(r.p * (double)m), s);
        }
        for (int g = wave; g < segs; g += NW) {
            Lane16<TL> x;
            x.load(row, V, g);
            double w = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) w += stays(x.v[e], g * SEG + x.at(e));
            w = wave_sum(w);
            if (lane == 0) sums[g] = w;
        }
    } else if (!r.min) {  // (relative to its own maximum each)
        for (int g = threadIdx.x; g < segs; g += THREADS) sums[g] = sums[g] * weight_of(sc.seg_top[g], top, r.T);
    }
    __syncthreads();
    // the segment: up to 1024 of them at a time
    double total = 0;
    for (int g0 = 0; g0 < segs; g0 += THREADS) {
        double all;
        scan_before(g0 + (int)threadIdx.x < segs ? sums[g0 + threadIdx.x] : 0.0, s.part, &all);
        total += all;
    }
    const double want = u > 0.0 ? u * total : 0.0;
    __syncthreads();
    if (threadIdx.x == 0) s.pick = segs;
    __syncthreads();
    double run = 0;
    int last = -1;
    for (int g0 = 0; g0 < segs && s.pick == segs; g0 += THREADS) {  // (the same in all threads: a barrier lies between)
        double all;
        const int g = g0 + threadIdx.x;
        const double w = g < segs ? sums[g] : 0.0, before = run + scan_before(w, s.part, &all);
        run += all;
        if (w > 0.0) last = g;
        if (w > 0.0 && before + w > want) atomicMin(&s.pick, g);
        __syncthreads();
        if (g == s.pick) s.rest = want - before;
        __syncthreads();
    }
    // (nothing found: u is 1 or more, or the sums were rounded: the last token that stays)
    if (s.pick == segs) {
        __syncthreads();
        if (threadIdx.x == 0) s.pick = -1;
        s.rest = 1e300;
        __syncthreads();
        atomicMax(&s.pick, last);
        __syncthreads();
    }
    const int seg = s.pick;
    const double rest = s.rest;
    const int i = seg * SEG + threadIdx.x;
    double all;
    const double w = i < V ? stays(value_at(row, i), i) : 0.0, before = scan_before(w, s.part, &all);
    __syncthreads();
    if (threadIdx.x == 0) s.found = 0xffffffffu, s.bin = 0;
    __syncthreads();
    if (w > 0.0) {
        if (before + w > rest) atomicMin(&s.found, (uint32_t)i);
        atomicMax(&s.bin, (uint32_t)i);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.ids[row_at] = (int)(s.found != 0xffffffffu ? s.found : s.bin);
}

size_t sample_scratch_bytes(int B, int V) { return (size_t)B * row_bytes(V); }

template <typename TL>
static int launch(const SampleArgs& a, int B, hipStream_t st) {
    const int segs = (a.V + SEG - 1) / SEG, slices = (segs + SLICE - 1) / SLICE;
    // (what a number for all rows rules out is not launched)
    const bool greedy = (!a.temperature && !(a.temperature_all > 0.0)) || (!a.top_k && a.top_k_all == 1) || (!a.top_p && a.top_p_all <= 0.0);
    const bool open = !a.top_k && (a.top_k_all <= 0 || a.top_k_all >= a.V) && !a.top_p && a.top_p_all >= 1.0 && !a.min_p && a.min_p_all <= 0.0;
    hipLaunchKernelGGL(sample_slices_kernel<TL>, dim3((unsigned)slices, (unsigned)B), dim3(THREADS), 0, st, a);
    if (!greedy && !open) hipLaunchKernelGGL(sample_filter_kernel<TL>, dim3((unsigned)slices, (unsigned)B), dim3(THREADS), 0, st, a);
    hipLaunchKernelGGL(sample_draw_kernel<TL>, dim3((unsigned)B), dim3(THREADS), 0, st, a);
    return check_hip(hipGetLastError(), "sample_draw_kernel launch");
}
int launch_sample(const SampleArgs& a, int B, bool f32, hipStream_t st) { return f32 ? launch<float>(a, B, st) : launch<uint16_t>(a, B, st); }

}  // namespace mmx
