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
// Four kernels, or one for a short row (sample_row_kernel).  A workgroup for each slice of a row reads the logits: segments' maxima; without filters their sums too; with top_k or top_p a histogram of the slice, counts and weights by
// l / T in steps of 1 / 16, on one grid for the row.  With filters a workgroup a row adds the histograms up, which shows the bin in which the run ends.  Workgroups of four segments collect what lies in it
// and above; or, where that is more than a list holds, what lies in it, and the segments' sums of what lies above.  A workgroup a row sorts out from the list where the run ends, and draws.
// Bound: the launches and the steps that wait for each other in them (barriers, LDS, a dependent read), each kernel 5 us at the least.  For many rows without filters the weights beside memory: the one pass
// over 256 x 131072 fp32 takes 35 us of 42, 3.8 TB/s, and its vector instructions, 30 a logit, 17 of them in 64 bits, 0.69 of that; without weights, temperature 0, the whole draw takes 28.  min_p alone
// passes twice: 65.  us, slices / cut / filter / draw: 33 x 100003 fp32, top_p 9 / 5 / 13 / 13;
// 64 x 131072 bf16, a mixture 13 / 5 / 11 / 16.  (One kernel, a workgroup a row that passes over it again and again: 349 and 589 us for these two.)
// Rows that this does not suit are worked on by that one workgroup alone, a pass over the row for every eight bits of the key.  They are those with more than a list
//   below the grid, 31.9 T under the largest, where the run ends there (top_k at a low temperature: 64 x 131072 bf16 with a dozen peaks, top_k 50: T 0.8 29 us, 0.2 332; 1 x 32000 fp32 T 0.2 17, 0.1 82);
//   in the bin in which top_k ends and above it, if there is a top_p too, or more than 2^20 logits;
//   of equal logits where the run ends;
// and those of 2^26 bins and more (|l / T| from 2^22 on, +inf) or temperatures past 1e-299 and 1e31.
#include "sample.hpp"

#include "ffn.hpp"

namespace mmx {

int num_cus();

constexpr int SEG = 1024;                 // logits of a segment
constexpr int BINS = 512;                 // the last one: everything below, e^-31.9 of the largest weight or less, which top_p's run takes for nothing
constexpr double PER_UNIT = 16;           // bins of a unit of l / T
constexpr int LIST = 4096;                // entries
constexpr int MOST_SLICES = 256;          // of a row
static_assert(MOST_SLICES * 16 * SEG == 1 << 22, "the longest row, in slices of sixteen segments");
constexpr int MOST_SUMS = 1024;           // segments of a row whose sums fit beside a list
constexpr double GRID = 67108864.0;        // 2^26: up to here what lies behind a bin's point is good to 2^-27
constexpr float NEVER = -__builtin_huge_valf();

// What a row asks for
struct RowAsks {
    double T, per, p, min_p;  // per: 1 / T
    int k;
    bool greedy, top_k, top_p, min;
    __device__ __forceinline__ bool filtered() const { return !greedy && (top_k || top_p); }
};
__device__ __forceinline__ RowAsks asks_of(const SampleArgs& a, int row) {
    RowAsks r;
    r.T = a.temperature ? (double)a.temperature[row] : a.temperature_all;
    r.per = 1.0 / fmax(r.T, 1e-300);  // (that and less: any two logits that differ are too far apart for a weight; 1 / T must stay a number)
    r.k = a.top_k ? a.top_k[row] : a.top_k_all;
    r.p = a.top_p ? (double)a.top_p[row] : a.top_p_all;
    r.min_p = a.min_p_all;
    if (a.min_p) r.min_p = a.min_p[row] > 1.0f ? 1.0 : (double)a.min_p[row];  // (not fmin, which would lose a NaN; with more than 1, tokens whose weight comes out as 1 at a high temperature would fall)
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
// A list's entry: the key, of bf16 without the half that they have in common, above as many bits as V has of the complement of the index.  So entries are ordered like the tokens, none is 0, and equal
// or neighbouring keys lie as close as their indexes allow, which is what a search by ranges goes by (with the index in 32 bits below 32 of key, bf16's equal logits all fell into one bucket's counter).
template <typename TL>
__device__ __forceinline__ unsigned long long entry_of(float x, int i, int V) {
    const int bits = 32 - __clz(V);
    return (unsigned long long)(key_of(x) >> (sizeof(TL) == 2 ? 16 : 0)) << bits | ((1u << bits) - 1u - (uint32_t)i);
}
__device__ __forceinline__ unsigned long long order_of(unsigned long long c, int V) { return c & ((1u << (32 - __clz(V))) - 1u); }  // (falls where the index rises; 1 at the least)
__device__ __forceinline__ int index_of(unsigned long long c, int V) { return (int)((1u << (32 - __clz(V))) - 1u - (uint32_t)order_of(c, V)); }
template <typename TL>
__device__ __forceinline__ uint32_t key_in(unsigned long long c, int V) {
    const uint32_t k = (uint32_t)(c >> (32 - __clz(V)));
    return sizeof(TL) == 2 ? k << 16 | (k & 0x8000u ? 0u : 0xffffu) : k;
}
__device__ __forceinline__ float settled(float x) { return x != x ? NEVER : x + 0.0f; }

// 2^y for y <= 0: 2^n times the series of 2^f = e^(f ln 2) to its tenth power, |f| <= 1 / 2, whose rest is (ln 2 / 2)^11 / 11! = 2e-13.  n comes out of adding a number so large that
// nothing is left behind the point.  (The library's exp, with a division by the temperature, took most of the time: 256 rows of 131072 62 us in the first kernel.)
__device__ __forceinline__ double exp2_of(double y) {
    y = fmax(y, -2000.0);  // (NaN too)
    const double big = 6755399441055744.0;  // 1.5 * 2^52
    const double t = y + big, f = y - (t - big);
    constexpr double L = 0.6931471805599453094;
    constexpr double L2 = L * L, L4 = L2 * L2, L8 = L4 * L4;
    double p = L8 * L2 / 3628800;
    p = __builtin_fma(p, f, L8 * L / 362880);
    p = __builtin_fma(p, f, L8 / 40320);
    p = __builtin_fma(p, f, L4 * L2 * L / 5040);
    p = __builtin_fma(p, f, L4 * L2 / 720);
    p = __builtin_fma(p, f, L4 * L / 120);
    p = __builtin_fma(p, f, L4 / 24);
    p = __builtin_fma(p, f, L2 * L / 6);
    p = __builtin_fma(p, f, L2 / 2);
    p = __builtin_fma(p, f, L);
    p = __builtin_fma(p, f, 1.0);
    return ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, t));
}
constexpr double LOG2_E = 1.4426950408889634074;
__device__ __forceinline__ double exp_of(double x) { return exp2_of(x * LOG2_E); }
// per: 1 / temperature
__device__ __forceinline__ double weight_below(float l, float top, double per) {  // (of a top that is finite; -inf comes out as zero)
    return exp2_of(((double)l - (double)top) * (per * LOG2_E));  // (the difference first: of products it would be off by what is left of theirs, without bound for large logits)
}
__device__ __forceinline__ double weight_of(float l, float top, double per) {
    const double w = weight_below(l, top, per);
    return l == top ? 1.0 : l == NEVER ? 0.0 : w;  // (an infinite one too: the others have no weight beside it)
}

__device__ __forceinline__ float value_at(const uint16_t* row, int64_t i) { return settled(from_bf16(row[i])); }
__device__ __forceinline__ float value_at(const float* row, int64_t i) { return settled(row[i]); }

// The 16 values of a lane in a segment and where in the segment they lie: pieces of 16 bytes, a wavefront's one behind the other.
template <typename TL>
struct Lane16 {
    static constexpr int PER = 16 / (int)sizeof(TL);  // values of a piece
    float v[16];
    u32x4 w[16 / PER];  // as they are in memory, so that several segments can be on their way
    bool whole;
    __device__ __forceinline__ static int at(int e) { return (e / PER) * (64 * PER) + (threadIdx.x & 63) * PER + e % PER; }
    __device__ __forceinline__ void ask(const TL* row, int V, int seg) {
        const int64_t base = (int64_t)seg * SEG;
        whole = base + SEG <= V;
        if (whole) {
#pragma unroll
            for (int c = 0; c < 16 / PER; c++) __builtin_memcpy(&w[c], __builtin_assume_aligned(row + base + at(c * PER), sizeof(TL)), 16);  // (the hardware takes any address)
        }
    }
    __device__ __forceinline__ void get(const TL* row, int V, int seg) {
        const int64_t base = (int64_t)seg * SEG;
        if (whole) {
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
    __device__ __forceinline__ void load(const TL* row, int V, int seg) {
        ask(row, V, seg);
        get(row, V, seg);
    }
};

// Neighbours' values within a wavefront, by the register file's own paths (through LDS, as a general exchange goes, a sum of 64-bit values over a wavefront and its workgroup took 1.7 us in place of 0.9).
// A lane that has no such neighbour gets `none`.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T neighbour(T none, T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const uint64_t n = __builtin_bit_cast(uint64_t, none), x = __builtin_bit_cast(uint64_t, v);
        const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)n, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
        const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp((int)(n >> 32), (int)(x >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (uint64_t)high << 32 | low);
    }
}
constexpr int SHR_1 = 0x111, SHR_2 = 0x112, SHR_4 = 0x114, SHR_8 = 0x118, ROW_TO_NEXT = 0x142, HALF_TO_NEXT = 0x143;  // (rows of 16 lanes; a row's last lane to the next row, lane 31 to the upper half)
constexpr int XOR_1 = 0xb1, XOR_2 = 0x4e, MIRROR_8 = 0x141;
// a lane's value, for all
template <typename T>
__device__ __forceinline__ T of_lane(T v, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const uint64_t x = __builtin_bit_cast(uint64_t, v);
        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane), high = (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane);
        return __builtin_bit_cast(T, (uint64_t)high << 32 | low);
    }
}
// the sum over the lanes up to this one
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    const T zero = 0;
    v += neighbour<SHR_1, 0xf>(zero, v);
    v += neighbour<SHR_2, 0xf>(zero, v);
    v += neighbour<SHR_4, 0xf>(zero, v);
    v += neighbour<SHR_8, 0xf>(zero, v);
    v += neighbour<ROW_TO_NEXT, 0xa>(zero, v);
    v += neighbour<HALF_TO_NEXT, 0xc>(zero, v);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    return of_lane(wave_scan(v), 63);
}
template <typename T>
__device__ __forceinline__ T larger(T a, T b) {
    return a > b ? a : b;
}
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
    v = larger(v, neighbour<SHR_1, 0xf>(v, v));
    v = larger(v, neighbour<SHR_2, 0xf>(v, v));
    v = larger(v, neighbour<SHR_4, 0xf>(v, v));
    v = larger(v, neighbour<SHR_8, 0xf>(v, v));
    v = larger(v, neighbour<ROW_TO_NEXT, 0xa>(v, v));
    v = larger(v, neighbour<HALF_TO_NEXT, 0xc>(v, v));
    return of_lane(v, 63);
}

// Of a number from each of up to sixteen wavefronts: what those before this one come to, and all of them.  (A lane reads one number; every lane reading all sixteen kept the LDS busy for half a
// microsecond.)
template <int WAVES, typename T>
__device__ __forceinline__ T of_waves(const T* part, T* all) {
    static_assert(WAVES <= 16, "a row of lanes");
    const int at = threadIdx.x & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T zero = 0;
    T v = at < WAVES ? part[at] : zero;
    v += neighbour<SHR_1, 0xf>(zero, v);
    v += neighbour<SHR_2, 0xf>(zero, v);
    v += neighbour<SHR_4, 0xf>(zero, v);
    v += neighbour<SHR_8, 0xf>(zero, v);
    *all = of_lane(v, 15);
    return wave > 0 ? of_lane(v, wave - 1) : zero;
}

constexpr int NW = 16, THREADS = NW * 64;

struct Cut {       // what stays: keys above, and of the equal ones indexes up to `index`
    uint32_t key;
    int index;
    __device__ __forceinline__ bool holds(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

// What a slice's workgroup leaves beside its histogram
struct Slice {
    double bin;  // of its largest logit
    uint32_t count, pad;
};
// Weights by bins: l / T = (bin + f) / PER_UNIT with f in [0, 1), so a weight is e^(f / PER_UNIT) times what all of the bin have in common.  A bin's word has its count above bit 49 and the sum
// of those factors, at most 1.065 each, as whole numbers of 2^-34 below (up to 2^14 of them).
constexpr int MASS_BITS = 49;
constexpr double FACTOR_SCALE = 17179869184.0;  // 2^34
// e^(f / 16) - 1 for f from [0, 1): the series to its seventh power, the rest is 6e-15
__device__ __forceinline__ double factor_less_1(double f) {
    const double x = f * (1.0 / PER_UNIT);
    double p = 1.0 / 5040;
    p = __builtin_fma(p, x, 1.0 / 720);
    p = __builtin_fma(p, x, 1.0 / 120);
    p = __builtin_fma(p, x, 1.0 / 24);
    p = __builtin_fma(p, x, 1.0 / 6);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    return p * x;
}
enum { BY_LIST, BY_SUMS, ALONE };
struct State {
    uint32_t entries, path, before_count;
    float top, from, to;       // logits from `from` on go into the list, those from `to` on into the sums
    double before_mass, mass;  // of what lies above the last bin, and of everything (0: it is not known, or all in the list)
};
// A row's scratch
struct Scratch {
    float* seg_top;
    double* sums;
    Slice* slices;
    State* state;
    unsigned long long* list;
    unsigned long long* bins;  // histograms, a slice's behind the other
    int segs, slice, n_slices;
};
__host__ __device__ inline size_t row_bytes(int V, int slice) {
    const size_t segs = ((size_t)V + SEG - 1) / SEG, slices = (segs + slice - 1) / slice;
    return (segs * 12 + slices * (sizeof(Slice) + BINS * 8) + LIST * 8 + sizeof(State) + 255) & ~(size_t)255;
}
__device__ __forceinline__ Scratch scratch_of(const SampleArgs& a, int row) {
    Scratch r;
    r.segs = (a.V + SEG - 1) / SEG;
    r.slice = a.slice;
    r.n_slices = (r.segs + r.slice - 1) / r.slice;
    char* p = a.scratch + (int64_t)row * row_bytes(a.V, r.slice);
    r.list = reinterpret_cast<unsigned long long*>(p), p += LIST * 8;
    r.state = reinterpret_cast<State*>(p), p += sizeof(State);
    r.slices = reinterpret_cast<Slice*>(p), p += r.n_slices * sizeof(Slice);
    r.bins = reinterpret_cast<unsigned long long*>(p), p += (int64_t)r.n_slices * BINS * 8;
    r.sums = reinterpret_cast<double*>(p), p += (int64_t)r.segs * 8;
    r.seg_top = reinterpret_cast<float*>(p);
    return r;
}
static_assert(sizeof(Slice) % 8 == 0 && sizeof(State) % 8 == 0 && MOST_SLICES <= BINS, "what lies behind them stays aligned; a slice a thread");

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
template <int WAVES = NW>
__device__ __forceinline__ double scan_before(double v, double* part, double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double run = wave_scan(v);
    __syncthreads();
    if (lane == 63) part[wave] = run;
    __syncthreads();
    return of_waves<WAVES>(part, all) + run - v;
}

// The cut that keeps the first `want_count` of what `limit` holds (by_mass: the shortest run of it that holds `want_mass`): its key by eight bits at a time from the top, over the whole row each time,
// then, if not all of the equal keys stay, the index.  Masses are whole numbers of 2^-shift, whose sums do not depend on their order.
template <typename TL>
__device__ Cut select(const TL* row, int V, float top, double per, double scale, Cut limit, bool by_mass, uint32_t want_count, unsigned long long want_mass, Shared& s) {
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
                if (by_mass) atomicAdd(&s.mass[k >> shift & 255], whole(weight_of(x.v[e], top, per), scale));
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
        const unsigned long long each = whole(weight_of(of_key(prefix), top, per), scale);
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
// (the first thread whose condition holds, as a ballot a wavefront: atomics of all lanes on one word took 20 cycles a lane)
__device__ __forceinline__ void first_of(bool holds, uint32_t* first) {
    const uint64_t m = __ballot(holds);
    if (m && (threadIdx.x & 63) == 0) atomicMin(first, (uint32_t)(threadIdx.x + __builtin_ctzll(m)));
}
__device__ __forceinline__ void last_of(bool holds, uint32_t* last) {
    const uint64_t m = __ballot(holds);
    if (m && (threadIdx.x & 63) == 0) atomicMax(last, (uint32_t)(threadIdx.x + 63 - __builtin_clzll(m)));
}

// SLICE wavefronts, a segment each
template <typename TL, int SLICE>
__global__ __launch_bounds__(SLICE * 64) __attribute__((amdgpu_waves_per_eu(8, 8))) void sample_slices_kernel(const SampleArgs a) {
    constexpr int WG = SLICE * 64;
    __shared__ unsigned long long bins[BINS];
    __shared__ uint32_t last;
    __shared__ double part[SLICE];
    __shared__ float tops[SLICE];
    __shared__ uint32_t counts[SLICE];
    const int row_at = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Scratch sc = scratch_of(a, row_at);
    const int g = blockIdx.x * SLICE + wave;
    const bool here = g < sc.segs;
    Lane16<TL> x;
    if (here) x.load(reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld), a.V, g);
    const RowAsks r = asks_of(a, row_at);
    float mine = NEVER;
    if (here) {
#pragma unroll
        for (int e = 0; e < 16; e++) mine = fmaxf(mine, x.v[e]);
    }
    float top = wave_max(mine);
    if (here && lane == 0) sc.seg_top[g] = top;
    if (!r.filtered()) {
        if (!here || r.greedy || r.min) return;
        double w = 0;
        if (top < __builtin_huge_valf()) {
#pragma unroll
            for (int e = 0; e < 16; e++) w += weight_below(x.v[e], top, r.per);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) w += x.v[e] == top ? 1.0 : 0.0;
        }
        w = wave_sum(top == NEVER ? 0.0 : w);
        if (lane == 0) sc.sums[g] = w;
        return;
    }
    if (lane == 0) tops[wave] = top;
    for (int i = threadIdx.x; i < BINS; i += WG) bins[i] = 0;
    if (threadIdx.x == 0) last = BINS;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SLICE; w++) top = fmaxf(top, tops[w]);
    const double per = PER_UNIT * r.per, bin = floor((double)top * per);
    auto bin_of = [&](double t) __attribute__((always_inline)) {
        const double d = bin - t;
        return d < BINS - 1 ? (int)d : BINS - 1;  // (NaN too: the last)
    };
    int until = BINS;  // bins from here on are of no interest
    if (r.top_k && r.k <= WG) {
        // The lanes' maxima alone: where k of them lie is a bin below which nothing can be among the first k.
        if (mine != NEVER) atomicAdd(&bins[bin_of(floor((double)mine * per))], 1ull);
        __syncthreads();
        constexpr int EACH = BINS / WG > 0 ? BINS / WG : 1;
        double n[EACH], all, sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int b = threadIdx.x * EACH + i;
            n[i] = b < BINS ? (double)bins[b] : 0.0;
            sum += n[i];
        }
        double run = scan_before<SLICE>(sum, part, &all);
        bool enough = false;
        uint32_t at = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            run += n[i];
            if (!enough && run >= (double)r.k) enough = true, at = threadIdx.x * EACH + i;
        }
        const uint64_t m = __ballot(enough && threadIdx.x * EACH < BINS);
        const uint32_t first = of_lane(at, m ? __builtin_ctzll(m) : 0);
        if (m && lane == 0) atomicMin(&last, first);
        __syncthreads();
        until = (int)last + 1;
        for (int i = threadIdx.x; i < BINS; i += WG) bins[i] = 0;
        __syncthreads();
    }
    uint32_t n = 0;
    if (top != NEVER && here) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const double t = (double)x.v[e] * per, low = floor(t);
            const int at = bin_of(low);
            if (x.v[e] == NEVER) continue;
            n++;
            if (at >= until) continue;
            unsigned long long w = 1ull << MASS_BITS;
            if (!r.top_k) w += (1ull << 34) + (uint32_t)(factor_less_1(t - low) * FACTOR_SCALE + 0.5);  // (top_k goes by counts)
            atomicAdd(&bins[at], w);
        }
    }
    n = wave_sum(n);
    if (lane == 0) counts[wave] = n;
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += WG) sc.bins[(int64_t)blockIdx.x * BINS + i] = bins[i];
    if (threadIdx.x == 0) {
        uint32_t all = 0;
#pragma unroll
        for (int w = 0; w < SLICE; w++) all += counts[w];
        sc.slices[blockIdx.x] = Slice{bin, all, 0};
    }
}

// ---- what the filters leave ---------------------------------------------------------------------------
// the largest of all (first: this thread's own of the row's segments' maxima)
template <int WAVES>
__device__ __forceinline__ float row_top(const Scratch& sc, float first, float* part) {
    float top = first;
    for (int i = WAVES * 64 + threadIdx.x; i < sc.segs; i += WAVES * 64) top = fmaxf(top, sc.seg_top[i]);
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, part[w]);
    return top;
}

// the least logit whose bin is `at` or more
__device__ __forceinline__ float least_of(double at, double per) {
    uint32_t k = key_of(settled((float)(at / per)));
    while (floor((double)of_key(k) * per) >= at) k--;
    while (floor((double)of_key(k) * per) < at) k++;
    return settled(of_key(k));
}

// the row's histogram, a bin a thread, and the bin in which the run ends.  A bin of more than a list holds (flat rows of large vocabularies) is cut into PARTS of its own first, for which the workgroup
// reads the row: 8 x 262144 fp32 of N(0, 1), top_p 0.9, 157 us in place of the 632 of one workgroup and the whole key.
// (A function of T threads, BINS or more, that all call; counts and masses_of: PARTS each.)
constexpr int PARTS = 2 * BINS;
template <typename TL, int T>
__device__ __forceinline__ void find_cut(const SampleArgs& a, const Scratch& sc, const RowAsks& r, int row_at, uint32_t* counts, unsigned long long* masses_of) {
    constexpr int WAVES = T / 64, AHEAD = 8;
    __shared__ State shared;
    __shared__ bool narrow;
    __shared__ uint32_t cpart[WAVES], first_part, last_part;
    __shared__ unsigned long long mpart[WAVES];
    __shared__ double part[2][WAVES];
    __shared__ int slice_ahead[MOST_SLICES];
    __shared__ float fpart[WAVES];
    __shared__ uint32_t found, last_bin, all_count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = threadIdx.x;
    const float first_top = b < sc.segs ? sc.seg_top[b] : NEVER;
    Slice own = {0.0, 0, 0};
    if (b < sc.n_slices) own = sc.slices[b];
    if (b == 0) found = BINS, last_bin = 0, all_count = 0, first_part = PARTS, last_part = 0;
    const float top = row_top<WAVES>(sc, first_top, fpart);
    if (top == NEVER) {
        if (b == 0) sc.state->path = ALONE;
        return;
    }
    const double per = PER_UNIT * r.per, at0 = (double)top * per, bin = floor(at0);
    const bool odd = !(fabs(bin) <= GRID) || !(per <= 1e300) || per < 1e-30;
    if (b < sc.n_slices) {
        // (a slice that lies below the grid, or holds nothing, has nothing in the row's other bins)
        const double ahead = bin - own.bin;
        slice_ahead[b] = ahead < BINS ? (int)ahead : BINS;
    }
    const uint32_t held = wave_sum(own.count);
    if (lane == 0 && held) atomicAdd(&all_count, held);
    __syncthreads();
    unsigned long long masses = 0;
    uint32_t count = 0;
    if (!odd) {
        for (int i0 = 0; i0 < sc.n_slices; i0 += AHEAD) {  // (AHEAD slices' bins on their way together)
            unsigned long long v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int at = i0 + i < sc.n_slices && b < BINS - 1 ? b - slice_ahead[i0 + i] : -1;
                v[i] = at >= 0 ? sc.bins[(int64_t)(i0 + i) * BINS + at] : 0ull;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                masses += v[i] & ((1ull << MASS_BITS) - 1);
                count += (uint32_t)(v[i] >> MASS_BITS);
            }
        }
    }
    const double mass = r.top_k ? 0.0 : (double)masses / FACTOR_SCALE * exp_of((bin - b - at0) * (1.0 / PER_UNIT));
    double run_mass = wave_scan(mass);
    uint32_t run_count = wave_scan(count);
    if (lane == 63) part[0][wave] = run_mass, part[1][wave] = run_count;
    __syncthreads();
    double all_mass, counted;
    run_mass += of_waves<WAVES>(part[0], &all_mass);
    run_count += (uint32_t)of_waves<WAVES>(part[1], &counted);
    if (b == BINS - 1) count = all_count - run_count, run_count = all_count;
    // of top_k the first whose count is enough, of top_p alone the first whose mass is (of both: top_p's share is of what top_k leaves, which only the list tells)
    first_of(r.top_k ? run_count >= (uint32_t)r.k : run_mass >= r.p * all_mass, &found);
    last_of(count > 0, &last_bin);
    __syncthreads();
    const int cut = found < BINS ? (int)found : (int)last_bin;  // (none: fewer tokens than top_k, or sums that were rounded)
    if (b == cut) {
        State s;
        s.entries = 0, s.before_count = run_count - count, s.top = top, s.before_mass = run_mass - mass, s.mass = all_mass;
        s.path = odd ? ALONE : run_count <= LIST ? BY_LIST : (r.top_k && r.top_p) || sc.segs > MOST_SUMS || (count > LIST && cut == BINS - 1) ? ALONE : BY_SUMS;
        s.from = s.to = __builtin_huge_valf();
        if (s.path != ALONE) {
            s.from = cut == BINS - 1 ? of_key(key_of(NEVER) + 1) : least_of(bin - cut, per);
            if (s.path == BY_SUMS && cut > 0) s.to = least_of(bin - cut + 1, per);
        }
        // (0: all there is lies in the list, whose own sum tells whether a share of it is reached; the histogram's, rounded otherwise, would have two equal logits and top_p 0.5 keep both)
        if (s.path == BY_LIST && (double)run_count >= counted) s.mass = 0.0;
        narrow = s.path == BY_SUMS && count > LIST;
        if (narrow) shared = s;
        else *sc.state = s;
    }
    for (int i = b; i < PARTS; i += T) counts[i] = 0, masses_of[i] = 0;
    __syncthreads();
    if (!narrow) return;
    State s = shared;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    const float low = s.from, high = cut > 0 ? s.to : top, each = (float)PARTS / (high - low);
    const double scale = (double)(1ull << a.shift);
    auto part_of = [&](float l) __attribute__((always_inline)) {  // (rises with l; a bin of one value: 0)
        const float x = (l - low) * each;
        return x >= PARTS - 1 ? PARTS - 1 : x > 0.0f ? (int)x : 0;
    };
    constexpr int TOGETHER = T == BINS ? 4 : 1;  // segments of a wavefront (as far as the registers go)
    for (int g0 = wave; g0 < sc.segs; g0 += WAVES * TOGETHER) {
        Lane16<TL> x[TOGETHER];
        bool some[TOGETHER];
#pragma unroll
        for (int t = 0; t < TOGETHER; t++) {
            const int g = g0 + t * WAVES;
            some[t] = g < sc.segs && sc.seg_top[g] >= low;
            if (some[t]) x[t].ask(row, a.V, g);
        }
#pragma unroll
        for (int t = 0; t < TOGETHER; t++) {
            if (!some[t]) continue;
            x[t].get(row, a.V, g0 + t * WAVES);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float l = x[t].v[e];
                if (l < low || l >= s.to) continue;
                const int at = part_of(l);
                atomicAdd(&counts[at], 1u);
                if (!r.top_k) atomicAdd(&masses_of[at], whole(weight_of(l, top, r.per), scale));
            }
        }
    }
    __syncthreads();
    // two parts a thread, in descending order
    uint32_t n[2] = {0, 0};
    unsigned long long m[2] = {0, 0};
    if (b < BINS) {
#pragma unroll
        for (int i = 0; i < 2; i++) n[i] = counts[PARTS - 1 - i - 2 * b], m[i] = masses_of[PARTS - 1 - i - 2 * b];
    }
    uint32_t c_run = wave_scan(n[0] + n[1]), c_all;
    unsigned long long m_run = wave_scan(m[0] + m[1]), m_all;
    if (lane == 63) cpart[wave] = c_run, mpart[wave] = m_run;
    __syncthreads();
    c_run += of_waves<WAVES>(cpart, &c_all) - n[0] - n[1];  // (what lies above the first of the two)
    m_run += of_waves<WAVES>(mpart, &m_all) - m[0] - m[1];
    auto reaches = [&](uint32_t c, unsigned long long w) __attribute__((always_inline)) { return r.top_k ? s.before_count + c >= (uint32_t)r.k : s.before_mass + (double)w / scale >= r.p * s.mass; };
    const int here = n[0] && reaches(c_run + n[0], m_run + m[0]) ? 2 * b : n[1] && reaches(c_run + n[0] + n[1], m_run + m[0] + m[1]) ? 2 * b + 1 : -1, held_here = n[1] ? 2 * b + 1 : n[0] ? 2 * b : -1;
    {
        const uint64_t hits = __ballot(here >= 0), any = __ballot(held_here >= 0);
        const int first = of_lane(here, hits ? __builtin_ctzll(hits) : 0), end = of_lane(held_here, any ? 63 - __builtin_clzll(any) : 0);
        if (lane == 0) {
            if (hits) atomicMin(&first_part, (uint32_t)first);
            if (any) atomicMax(&last_part, (uint32_t)end);
        }
    }
    __syncthreads();
    const int at = first_part < PARTS ? (int)first_part : (int)last_part;
    if (b != at >> 1) return;
    const bool second = at & 1;
    const uint32_t entries = second ? n[1] : n[0];
    s.before_count += c_run + (second ? n[0] : 0u);
    s.before_mass += (double)(m_run + (second ? m[0] : 0ull)) / scale;
    if (entries > LIST) s.path = ALONE;
    auto least_in = [&](int q) __attribute__((always_inline)) {  // the least logit of part q or a higher one
        uint32_t from = key_of(low), to = key_of(high);
        while (from < to) {
            const uint32_t mid = from + (to - from) / 2;
            if (part_of(of_key(mid)) >= q) to = mid;
            else from = mid + 1;
        }
        return of_key(from);
    };
    const int q = PARTS - 1 - at;
    if (q < part_of(high)) s.to = least_in(q + 1);
    s.from = least_in(q);
    *sc.state = s;
}
template <typename TL>
__global__ __launch_bounds__(BINS) void sample_cut_kernel(const SampleArgs a) {
    __shared__ uint32_t counts[PARTS];
    __shared__ unsigned long long masses_of[PARTS];
    const RowAsks r = asks_of(a, blockIdx.x);
    if (r.filtered()) find_cut<TL, BINS>(a, scratch_of(a, blockIdx.x), r, blockIdx.x, counts, masses_of);
}

template <typename TL>
__global__ __launch_bounds__(256) void sample_filter_kernel(const SampleArgs a) {
    constexpr int WAVES = 4;
    __shared__ float fpart[WAVES];
    __shared__ uint32_t base, taken[WAVES];
    const int row_at = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Scratch sc = scratch_of(a, row_at);
    const int g = blockIdx.x * WAVES + wave;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    const bool here = g < sc.segs;
    // (everything that does not wait for something else first)
    const State state = *sc.state;
    const float seg_top = here ? sc.seg_top[g] : NEVER;
    const RowAsks r = asks_of(a, row_at);
    if (r.greedy || !(r.filtered() || r.min)) return;
    float top = state.top;
    Lane16<TL> x;
    if (!r.filtered()) {
        if (here) x.ask(row, a.V, g);
        top = row_top<WAVES>(sc, (int)threadIdx.x < sc.segs ? sc.seg_top[threadIdx.x] : NEVER, fpart);
        if (top == NEVER || !here) return;
    } else if (state.path == ALONE) {
        return;
    }
    auto weight = [&](float l) __attribute__((always_inline)) {
        const double v = weight_of(l, top, r.per);
        return v < r.min_p && l != top ? 0.0 : v;
    };
    if (!r.filtered()) {
        double w = 0;
        if (seg_top != NEVER) {
            x.get(row, a.V, g);
#pragma unroll
            for (int e = 0; e < 16; e++) w += weight(x.v[e]);
            w = wave_sum(w);
        }
        if (lane == 0) sc.sums[g] = w;
        return;
    }
    uint32_t takes = 0;
    const bool some = here && seg_top >= state.from;
    if (some) {
        x.ask(row, a.V, g);
        x.get(row, a.V, g);
    }
    if (state.path == BY_SUMS && here) {
        double w = 0;
        if (some && seg_top >= state.to) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (__any(x.v[e] >= state.to)) w += x.v[e] >= state.to ? weight(x.v[e]) : 0.0;
            w = wave_sum(w);
        }
        if (lane == 0) sc.sums[g] = w;
    }
    if (some) {
#pragma unroll
        for (int e = 0; e < 16; e++) takes |= x.v[e] >= state.from && x.v[e] < state.to ? 1u << e : 0;
    }
    const uint32_t mine = __popc(takes);
    uint32_t at = wave_scan(mine);
    if (lane == 63) taken[wave] = at;
    __syncthreads();
    uint32_t every = 0, before = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        before += i < wave ? taken[i] : 0;
        every += taken[i];
    }
    if (every == 0) return;
    if (threadIdx.x == 0) base = atomicAdd(&sc.state->entries, every);
    __syncthreads();
    at += base + before - mine;
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (takes >> e & 1) {
            if (at < LIST) sc.list[at] = entry_of<TL>(x.v[e], g * SEG + x.at(e), a.V);
            at++;
        }
}

// ---- where the run ends, a workgroup a row --------------------------------------------------------------------------------------------
constexpr int MINE = LIST / THREADS, BUCKETS = 1024, FEW = 128;
struct Room {
    unsigned long long mass[BUCKETS];
    uint32_t count[BUCKETS];
    __attribute__((aligned(16))) unsigned long long few[FEW][2];  // (with its mass)
    unsigned long long low, high, best, part[NW], before_mass;
    uint32_t cpart[NW], first, last;
};
static_assert(BUCKETS == PARTS, "a short row's cut borrows the buckets");
static_assert(BUCKETS == THREADS && FEW * 8 == THREADS, "a bucket a thread; eight threads for each that is left");

// Of the entries (a thread's c, no two alike; 0: none) in descending order: the first up to which there are `want` of them, or whose masses m come to `want` (STRICT: to more); the last if none does.
// The range of what is left is cut into 1024 buckets until one of them holds few, and those are compared with each other.
enum { BY_COUNT, BY_MASS, BY_MASS_STRICT };
// most: entries lie in the first `most` places.
__device__ __forceinline__ unsigned long long pick(const unsigned long long (&c)[MINE], const unsigned long long (&m)[MINE], int most, int mode, unsigned long long want, Room& o) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned long long low = 1, high = ~0ull, before = 0;  // of the entries from low to high; what lies above them
    int n = most;
    __syncthreads();  // (what an earlier call left has been read)
    if (most <= FEW) {
        if ((int)threadIdx.x < most) o.few[threadIdx.x][0] = c[0], o.few[threadIdx.x][1] = c[0] == 0 ? 0ull : mode == BY_COUNT ? 1ull : m[0];
        if (threadIdx.x == 0) o.best = 0, o.low = 0;
    }
    while (most > FEW) {
        unsigned long long lo = ~0ull, hi = 0;
        uint32_t here = 0;
#pragma unroll
        for (int i = 0; i < MINE; i++)
            if (i * THREADS < most && c[i] >= low && c[i] <= high) {
                here++;
                lo = c[i] < lo ? c[i] : lo;
                hi = c[i] > hi ? c[i] : hi;
            }
        const uint32_t at = wave_scan(here);
        __syncthreads();  // (what the last round left has been read)
        if (lane == 63) o.cpart[wave] = at;
        if (threadIdx.x == 0) o.low = ~0ull, o.high = 0, o.best = 0, o.first = BUCKETS, o.last = 0;
        __syncthreads();
        uint32_t every;
        uint32_t off = of_waves<NW>(o.cpart, &every) + at - here;
        n = (int)every;
        if (n <= FEW) {
#pragma unroll
            for (int i = 0; i < MINE; i++)
                if (i * THREADS < most && c[i] >= low && c[i] <= high) o.few[off][0] = c[i], o.few[off++][1] = mode == BY_COUNT ? 1ull : m[i];
            break;
        }
        if (__any(here)) {
            hi = wave_max(hi), lo = ~wave_max(~lo);
            if (lane == 0) {
                atomicMin(&o.low, lo);
                atomicMax(&o.high, hi);
            }
        }
        o.mass[threadIdx.x] = 0, o.count[threadIdx.x] = 0;
        __syncthreads();
        low = o.low, high = o.high;
        const unsigned long long span = high - low;
        const int bits = 64 - __clzll((long long)span), shift = bits > 10 ? bits - 10 : 0;
#pragma unroll
        for (int i = 0; i < MINE; i++)
            if (i * THREADS < most && c[i] >= low && c[i] <= high) {
                atomicAdd(&o.count[(high - c[i]) >> shift], 1u);
                if (mode != BY_COUNT) atomicAdd(&o.mass[(high - c[i]) >> shift], m[i]);
            }
        __syncthreads();
        const bool some = o.count[threadIdx.x] > 0;
        const unsigned long long mine = mode == BY_COUNT ? o.count[threadIdx.x] : o.mass[threadIdx.x];
        unsigned long long run = wave_scan(mine);
        if (lane == 63) o.part[wave] = run;
        __syncthreads();
        unsigned long long every_mass;
        run += of_waves<NW>(o.part, &every_mass) + before;
        first_of(some && (mode == BY_MASS_STRICT ? run > want : run >= want), &o.first);
        last_of(some, &o.last);
        __syncthreads();
        const int b = o.first < BUCKETS ? (int)o.first : (int)o.last;
        if ((int)threadIdx.x == b) o.before_mass = run - mine;
        __syncthreads();
        before = o.before_mass;
        const unsigned long long up = high - ((unsigned long long)b << shift), room = (1ull << shift) - 1;
        low = up - low > room ? up - room : low;
        high = up;
    }
    __syncthreads();
    // Eight neighbouring threads an entry, each against every eighth of them.  The one that is sought is the only one that reaches the goal and does not without its own mass.
    if ((int)(threadIdx.x & ~63u) < n * 8) {
        const int i = threadIdx.x >> 3;
        const unsigned long long mine = i < n ? o.few[i][0] : 0ull;
        unsigned long long run = 0;
        uint32_t after = 0;  // entries behind it
#pragma unroll 4
        for (int j = threadIdx.x & 7; j < n; j += 8) {
            const unsigned long long other = o.few[j][0], mass = o.few[j][1];
            run += other >= mine ? mass : 0ull;
            after += other < mine && other != 0 ? 1 : 0;
        }
        run += neighbour<XOR_1, 0xf>(0ull, run), after += neighbour<XOR_1, 0xf>(0u, after);
        run += neighbour<XOR_2, 0xf>(0ull, run), after += neighbour<XOR_2, 0xf>(0u, after);
        run += neighbour<MIRROR_8, 0xf>(0ull, run), after += neighbour<MIRROR_8, 0xf>(0u, after);  // (fours are alike by now)
        run += before;
        if (mine && (threadIdx.x & 7) == 0) {
            const unsigned long long less = run - o.few[i][1];
            if (mode == BY_MASS_STRICT ? run > want && less <= want : run >= want && less < want) o.best = mine;
            if (after == 0) o.low = mine;
        }
    }
    __syncthreads();
    return o.best ? o.best : o.low;
}
__device__ unsigned long long sum_of(unsigned long long v, Room& o) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) o.part[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long all;
    of_waves<NW>(o.part, &all);
    return all;
}

// A workgroup of THREADS for a row.  OWN: without filters, segments' sums are relative to their own maxima.
template <typename TL, bool OWN, int SUMS>
__device__ __forceinline__ void draw(const SampleArgs& a, const Scratch& sc, const RowAsks& r, int row_at, Shared& s, Room& o) {
    __shared__ unsigned long long more[SUMS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int V = a.V;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    const int segs = sc.segs;
    // (what the next steps want, asked for with the first)
    const State state = *sc.state;
    const double first_sum = (int)threadIdx.x < segs ? sc.sums[threadIdx.x] : 0.0;
    const float first_top = (int)threadIdx.x < segs ? sc.seg_top[threadIdx.x] : NEVER;
    const float asked = a.u[row_at];
    const double u = asked >= 1.0f ? __builtin_huge_val() : (double)asked;  // (nothing comes to 1 of the sum and more, but sums of another order may)
    unsigned long long c[MINE], m[MINE];
#pragma unroll
    for (int i = 0; i < MINE; i++) {  // (asked for before anything is known of it; sorted out below)
        c[i] = r.filtered() && i == 0 ? sc.list[threadIdx.x] : 0;
    }
    const bool known = r.filtered() && state.path != ALONE;  // (its largest logit)
    const float top = known ? state.top : row_top<NW>(sc, first_top, s.fpart);
    if (top == NEVER) {
        if (threadIdx.x == 0) a.ids[row_at] = -1;
        return;
    }
    if (r.greedy) {  // the first segment that holds it, its first place in it
        if (threadIdx.x == 0) s.pick = V, s.found = 0xffffffffu;
        __syncthreads();
        for (int g = threadIdx.x; g < segs; g += THREADS)
            if ((g < THREADS ? first_top : sc.seg_top[g]) == top) atomicMin(&s.pick, g);
        __syncthreads();
        const int seg = s.pick < segs ? s.pick : 0, i = seg * SEG + threadIdx.x;
        first_of(i < V && value_at(row, i) == top, &s.found);
        __syncthreads();
        if (threadIdx.x == 0) a.ids[row_at] = seg * SEG + (int)s.found;
        return;
    }
    const uint32_t path = r.filtered() ? state.path : BY_SUMS;
    const double scale = (double)(1ull << a.shift);
    Cut cut = {key_of(NEVER), V};
    auto stays = [&](float l, int i) __attribute__((always_inline)) {
        const double w = weight_of(l, top, r.per);
        return l == NEVER || !cut.holds(key_of(l), i) || (w < r.min_p && l != top) ? 0.0 : w;
    };
    if (r.filtered() && path != ALONE) {
        const int n = (int)state.entries < LIST ? (int)state.entries : LIST;
        unsigned long long last = 1;
        uint32_t low_weight = 0;
        const double least_p = fmax(r.min_p, 5e-324);  // (what 64 bits hold as 0 isn't drawn)
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const int at = threadIdx.x + i * THREADS;
            m[i] = 0;
            if (i * THREADS >= n) {
                c[i] = 0;
                continue;
            }
            if (i > 0) c[i] = at < n ? sc.list[at] : 0;
            if (at >= n) c[i] = 0;
            const float l = of_key(key_in<TL>(c[i], V));
            if (!__any(c[i] != 0)) continue;
            const double w = c[i] ? weight_of(l, top, r.per) : 0.0;
            m[i] = whole(w, scale);
            low_weight |= w < least_p && l != top ? 1u << i : 0;
        }
        const uint32_t above = path == BY_SUMS ? state.before_count : 0;
        for (int step = 0; step < 3; step++) {  // top_k, top_p, the token
            int mode = BY_COUNT;
            unsigned long long want = 0;
            if (step == 0) {
                if (!r.top_k || above + (uint32_t)n <= (uint32_t)r.k) continue;
                want = (uint32_t)r.k - above;
            } else if (step == 1) {  // (not BY_SUMS and top_k both)
                if (!r.top_p) continue;
                unsigned long long of = 0;
#pragma unroll
                for (int i = 0; i < MINE; i++) of += c[i] ? m[i] : 0ull;
                const bool own_sum = state.mass == 0.0;  // (always with top_k)
                if (own_sum) of = sum_of(of, o);
                const double goal = ceil(r.p * (own_sum ? (double)of : state.mass * scale)) - (path == BY_SUMS ? state.before_mass * scale : 0.0);
                mode = BY_MASS, want = goal > 1.0 ? (unsigned long long)goal : 1ull;
            } else {
                unsigned long long all = 0;
#pragma unroll
                for (int i = 0; i < MINE; i++) {
                    if (low_weight >> i & 1) c[i] = 0;
                    // (what stays can be drawn, by a u of 0 or 1, however small its weight; to top_p's share such weights add nothing, as in 64 bits)
                    m[i] = c[i] ? larger(m[i], 1ull) : 0ull;
                    all += m[i];
                    c[i] = order_of(c[i], V);  // (the order of the vocabulary)
                }
                if (path == BY_SUMS) break;
                all = sum_of(all, o);
                const double goal = u > 0.0 ? u * (double)all : 0.0;
                const bool inside = goal < (double)all;  // (else the last one that has weight)
                mode = inside ? BY_MASS_STRICT : BY_MASS, want = inside ? (unsigned long long)goal : all;
            }
            last = pick(c, m, n, mode, want, o);
            if (step < 2) {
#pragma unroll
                for (int i = 0; i < MINE; i++) c[i] = c[i] < last ? 0 : c[i];
            }
        }
        if (path == BY_LIST) {
            if (threadIdx.x == 0) a.ids[row_at] = index_of(last, V);
            return;
        }
        // what stays of the bin, to its segments' sums
        for (int g = threadIdx.x; g < segs; g += THREADS) more[g] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MINE; i++)
            if (c[i]) atomicAdd(&more[index_of(c[i], V) / SEG], m[i]);
        // (nothing was cut off the list where top_k ends with it: what lies below the list does not stay)
        cut = last > 1 ? Cut{key_in<TL>(last, V), index_of(last, V)} : Cut{key_of(state.from), V};
        __syncthreads();
    } else if (path == ALONE) {
        if (r.top_k) cut = select(row, V, top, r.per, scale, cut, false, (uint32_t)r.k, 0ull, s);
        if (r.top_p) {
            unsigned long long m = 0;
            for (int g = wave; g < segs; g += NW) {
                Lane16<TL> x;
                x.load(row, V, g);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (cut.holds(key_of(x.v[e]), g * SEG + x.at(e))) m += whole(weight_of(x.v[e], top, r.per), scale);
            }
            m = wave_sum(m);
            __syncthreads();
            if (lane == 0) s.mass[wave] = m;
            __syncthreads();
            m = 0;
            for (int w = 0; w < NW; w++) m += s.mass[w];
            cut = select(row, V, top, r.per, scale, cut, true, 0u, (unsigned long long)ceil(r.p * (double)m), s);
        }
        for (int g = wave; g < segs; g += NW) {
            Lane16<TL> x;
            x.load(row, V, g);
            double w = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) w += stays(x.v[e], g * SEG + x.at(e));
            w = wave_sum(w);
            if (lane == 0) sc.sums[g] = w;
        }
        __syncthreads();
    }
    // A segment's sum: without filters it is relative to its own maximum, with a list there may be more to it.  A thread has up to four neighbouring segments (of 2^22 logits).
    constexpr int MOST = 4;
    const bool own = OWN && !r.filtered() && !r.min, added = r.filtered() && path == BY_SUMS;
    const int each = (segs + THREADS - 1) / THREADS, g0 = threadIdx.x * each;
    double sums[MOST], mine = 0, total;
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        const int g = g0 + k;
        sums[k] = 0;
        if (k >= each || g >= segs) continue;
        const bool ready = each == 1 && path != ALONE;
        const double w = ready ? first_sum : sc.sums[g];
        sums[k] = own ? w * weight_of(ready ? first_top : sc.seg_top[g], top, r.per) : added ? w + (double)more[g] / scale : w;
        mine += sums[k];
    }
    if (threadIdx.x == 0) s.pick = segs, s.bin = 0;
    double run = scan_before(mine, s.part, &total);
    const double want = u > 0.0 ? u * total : 0.0;
    int here = -1, last = -1;
    double rest = 0;
#pragma unroll
    for (int k = 0; k < MOST; k++) {
        if (sums[k] > 0.0) {
            if (here < 0 && run + sums[k] > want) here = g0 + k, rest = want - run;
            last = g0 + k;
        }
        run += sums[k];
    }
    {
        const uint64_t m = __ballot(here >= 0), any = __ballot(last >= 0);
        const int first = of_lane(here, m ? __builtin_ctzll(m) : 0), end = of_lane(last, any ? 63 - __builtin_clzll(any) : 0);
        if (lane == 0) {
            if (m) atomicMin(&s.pick, first);
            if (any) atomicMax(&s.bin, (uint32_t)end);
        }
    }
    __syncthreads();
    // (nothing found: u is 1 or more, or the sums were rounded: the last token that stays)
    const int seg = s.pick < segs ? s.pick : (int)s.bin;
    if (here == seg) s.rest = rest;
    else if (s.pick == segs && threadIdx.x == 0) s.rest = 1e300;
    const int i = seg * SEG + threadIdx.x;
    const double w = i < V ? stays(value_at(row, i), i) : 0.0;
    __syncthreads();
    rest = s.rest;
    if (threadIdx.x == 0) s.found = 0xffffffffu, s.bin = 0;
    double all;
    const double before = scan_before(w, s.part, &all);
    first_of(w > 0.0 && before + w > rest, &s.found);
    last_of(w > 0.0, &s.bin);
    __syncthreads();
    if (threadIdx.x == 0) a.ids[row_at] = seg * SEG + (int)(s.found != 0xffffffffu ? s.found : s.bin);
}

template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_draw_kernel(const SampleArgs a) {
    __shared__ Shared s;
    __shared__ Room o;
    draw<TL, true, MOST_SUMS>(a, scratch_of(a, blockIdx.x), asks_of(a, blockIdx.x), blockIdx.x, s, o);
}

// ---- a short row in one workgroup ---------------------------------------------------------------------------------------------------
// The same steps with what they hand on in LDS, two segments a wavefront, read once: three launches less, and one CU's exponentials and LDS atomics in place of several's (the rule below).
constexpr int ROW_SEGS = 2 * NW;
template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(const SampleArgs a) {
    __shared__ Shared s;
    __shared__ Room o;
    __shared__ unsigned long long list[LIST], bins[2][BINS];  // (a histogram for eight wavefronts each: up to 2^14 logits)
    __shared__ State state;
    __shared__ Slice slices[2];
    __shared__ double sums[ROW_SEGS];
    __shared__ float seg_top[ROW_SEGS];
    const int row_at = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave / (NW / 2);
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    Scratch sc;
    sc.segs = (a.V + SEG - 1) / SEG, sc.slice = NW, sc.n_slices = 2;
    sc.seg_top = seg_top, sc.sums = sums, sc.slices = slices, sc.state = &state, sc.list = list, sc.bins = bins[0];
    const RowAsks r = asks_of(a, row_at);
    Lane16<TL> x[2];
#pragma unroll
    for (int t = 0; t < 2; t++)
        if (wave * 2 + t < sc.segs) x[t].ask(row, a.V, wave * 2 + t);
    bins[threadIdx.x / BINS][threadIdx.x % BINS] = 0;
    if (threadIdx.x < 2) slices[threadIdx.x].count = 0;
    if (threadIdx.x == 0) s.found = 0;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int g = wave * 2 + t;
        if (g >= sc.segs) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[t].v[e] = NEVER;
            continue;
        }
        x[t].get(row, a.V, g);
        float mine = NEVER;
#pragma unroll
        for (int e = 0; e < 16; e++) mine = fmaxf(mine, x[t].v[e]);
        mine = wave_max(mine);
        if (lane == 0) seg_top[g] = mine;
    }
    __syncthreads();
    const float top = wave_max((lane & (ROW_SEGS - 1)) < sc.segs ? seg_top[lane & (ROW_SEGS - 1)] : NEVER);
    auto weight = [&](float l) __attribute__((always_inline)) {
        const double v = weight_of(l, top, r.per);
        return v < r.min_p && l != top ? 0.0 : v;
    };
    if (top != NEVER && !r.greedy) {
        if (!r.filtered()) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                double w = 0;
#pragma unroll
                for (int e = 0; e < 16; e++) w += weight(x[t].v[e]);
                w = wave_sum(w);
                if (lane == 0 && wave * 2 + t < sc.segs) sums[wave * 2 + t] = w;
            }
        } else {
            const double per = PER_UNIT * r.per, bin = floor((double)top * per);
            double least = -__builtin_huge_val();  // what is smaller is of no interest
            if (r.top_k && r.k <= THREADS) {
                // the threads' largest alone: below the bin that the k-th of them lies in nothing can be among the first k (one bin more, for what is rounded here)
                float mine = NEVER;
#pragma unroll
                for (int e = 0; e < 16; e++) mine = fmaxf(mine, fmaxf(x[0].v[e], x[1].v[e]));
                const double d = bin - floor((double)mine * per);
                if (mine != NEVER && d < BINS - 1) atomicAdd(&bins[0][(int)d], 1ull);
                if (threadIdx.x == 0) s.bin = BINS;
                __syncthreads();
                const uint32_t held = threadIdx.x < BINS ? (uint32_t)bins[0][threadIdx.x] : 0u;
                const uint32_t run = wave_scan(held);
                if (lane == 63) o.cpart[wave] = run;
                __syncthreads();
                uint32_t all;
                first_of(of_waves<NW>(o.cpart, &all) + run >= (uint32_t)r.k, &s.bin);
                if (threadIdx.x < BINS) bins[0][threadIdx.x] = 0;
                __syncthreads();
                if (s.bin < BINS) least = (bin - (double)s.bin - 1.0) / per;
            }
            uint32_t n = 0;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    if (x[t].v[e] == NEVER) continue;
                    n++;
                    if ((double)x[t].v[e] < least) continue;
                    const double l = (double)x[t].v[e] * per, low = floor(l), d = bin - low;
                    unsigned long long w = 1ull << MASS_BITS;
                    if (!r.top_k) w += (1ull << 34) + (uint32_t)(factor_less_1(l - low) * FACTOR_SCALE + 0.5);
                    if (d < BINS - 1) atomicAdd(&bins[part][(int)d], w);  // (what lies in the last is counted only)
                }
            n = wave_sum(n);
            if (lane == 0) {
                if (n) atomicAdd(&slices[part].count, n);
                slices[part].bin = bin;
            }
            __syncthreads();
            find_cut<TL, THREADS>(a, sc, r, row_at, o.count, o.mass);
            __syncthreads();
            const State at = state;
            if (at.path != ALONE) {
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (at.path == BY_SUMS) {
                        double w = 0;
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (__any(x[t].v[e] >= at.to)) w += x[t].v[e] >= at.to ? weight(x[t].v[e]) : 0.0;
                        w = wave_sum(w);
                        if (lane == 0 && wave * 2 + t < sc.segs) sums[wave * 2 + t] = w;
                    }
                    uint32_t takes = 0;
#pragma unroll
                    for (int e = 0; e < 16; e++) takes |= x[t].v[e] >= at.from && x[t].v[e] < at.to ? 1u << e : 0;
                    if (!__any(takes != 0)) continue;
                    const uint32_t mine = __popc(takes), upto = wave_scan(mine);
                    uint32_t to = 0;
                    if (lane == 63) to = atomicAdd(&s.found, upto);
                    to = of_lane(to, 63) + upto - mine;
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (takes >> e & 1) {
                            if (to < LIST) list[to] = entry_of<TL>(x[t].v[e], (wave * 2 + t) * SEG + Lane16<TL>::at(e), a.V);
                            to++;
                        }
                }
                __syncthreads();
                if (threadIdx.x == 0) state.entries = s.found;
            }
        }
    } else if (threadIdx.x == 0) {
        state.path = ALONE;  // (no largest logit in it)
    }
    __syncthreads();
    draw<TL, false, ROW_SEGS>(a, sc, r, row_at, s, o);
}

// Segments of a slice: 4 where 16 would leave most of the chip idle (1 x 32000: 8 workgroups in place of 2); 16 elsewhere, since every slice's histogram is written and read
int sample_slice(int B, int V) {
    const int64_t segs = ((int64_t)V + SEG - 1) / SEG;
    return B * ((segs + 15) / 16) < 64 && segs <= 4 * MOST_SLICES ? 4 : 16;
}
size_t sample_scratch_bytes(int B, int V) { return (size_t)B * row_bytes(V, sample_slice(B, V)); }

template <typename TL, int SLICE>
static int launch(const SampleArgs& a, int B, hipStream_t st) {
    const int segs = (a.V + SEG - 1) / SEG, slices = (segs + SLICE - 1) / SLICE;
    // (what a number for all rows rules out is not launched)
    const bool greedy = (!a.temperature && !(a.temperature_all > 0.0)) || (!a.top_k && a.top_k_all == 1) || (!a.top_p && a.top_p_all <= 0.0);
    const bool open = !a.top_k && (a.top_k_all <= 0 || a.top_k_all >= a.V) && !a.top_p && a.top_p_all >= 1.0 && !a.min_p && a.min_p_all <= 0.0;
    const bool filters = a.top_k || (a.top_k_all > 0 && a.top_k_all < a.V) || a.top_p || a.top_p_all < 1.0;
    // (short rows: us in one workgroup / in four kernels, fp32, rows 1, 64, 256: 32000 top_k 50 and top_p 0.9 19 / 22, 21 / 26, 24 / 35; 8000 top_p 0.9 26 / 30, 28 / 33, 28 / 38.  Where every logit has a factor of
    // a weight to be computed, a row takes longer in one workgroup from some 12 segments on: 32000 top_p 0.9 36 / 27, 37 / 33, 41 / 49; and without filters two kernels are faster: 8000 14 / 10, 16 / 11, 16 / 13.
    // 1024 rows of 5000, top_p: 104 / 100.)
    const bool by_count = !a.top_k && a.top_k_all > 0 && a.top_k_all < a.V;
    if (!greedy && filters && (by_count ? segs <= ROW_SEGS : segs <= 12 && B <= 2 * num_cus())) {
        hipLaunchKernelGGL(sample_row_kernel<TL>, dim3((unsigned)B), dim3(THREADS), 0, st, a);
        return check_hip(hipGetLastError(), "sample_row_kernel launch");
    }
    if (greedy || !filters)  // (no histograms: small workgroups, of which more overlap)
        hipLaunchKernelGGL((sample_slices_kernel<TL, 4>), dim3((unsigned)((segs + 3) / 4), (unsigned)B), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((sample_slices_kernel<TL, SLICE>), dim3((unsigned)slices, (unsigned)B), dim3(SLICE * 64), 0, st, a);
    if (!greedy && filters) hipLaunchKernelGGL(sample_cut_kernel<TL>, dim3((unsigned)B), dim3(BINS), 0, st, a);
    if (!greedy && !open) hipLaunchKernelGGL(sample_filter_kernel<TL>, dim3((unsigned)((segs + 3) / 4), (unsigned)B), dim3(256), 0, st, a);
    hipLaunchKernelGGL(sample_draw_kernel<TL>, dim3((unsigned)B), dim3(THREADS), 0, st, a);
    return check_hip(hipGetLastError(), "sample_draw_kernel launch");
}
int launch_sample(SampleArgs a, int B, bool f32, hipStream_t st) {
    a.slice = sample_slice(B, a.V);
    if (a.slice == 4) return f32 ? launch<float, 4>(a, B, st) : launch<uint16_t, 4>(a, B, st);
    return f32 ? launch<float, 16>(a, B, st) : launch<uint16_t, 16>(a, B, st);
}

}  // namespace mmx
