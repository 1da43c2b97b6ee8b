// Drawing one token a row from logits l [B, V], given a random number u from [0, 1) for each row:
//
//   w_i = e^((l_i - max l) / T)                            weights in 64 bits; -inf and NaN have none
//   order: descending l, the lowest index of equal ones first
//   top_k: the first k of it stay; top_p: of those the shortest run that holds p of their weight at least; min_p: of those what has w >= min_p
//   the token: the first in the order of the vocabulary up to which the weights that stay come to more than u of their sum
//
// What stays is a run of the order whatever the filters are, so it is held as its last element: a key (the bits of l, made to order like l) and, among equal keys, an index.
// A row is cut into segments of 1024 neighbours, one wavefront's 16 values a lane, whose maxima and sums are what the draw goes by: it finds its segment, then its token in it.
#include "sample.hpp"

#include "ffn.hpp"

namespace mmx {

constexpr int SEG = 1024;
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

// ---- the one kernel: a workgroup of sixteen wavefronts a row ------------------------------------------------------------------
constexpr int NW = 16, THREADS = NW * 64;

struct Cut {       // what stays: keys above, and of the equal ones indexes up to `index`
    uint32_t key;
    int index;
    __device__ __forceinline__ bool holds(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

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
                if (by_mass) atomicAdd(&s.mass[k >> shift & 255], (unsigned long long)(weight_of(x.v[e], top, T) * scale + 0.5));
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
        const unsigned long long each = (unsigned long long)(weight_of(of_key(prefix), top, T) * scale + 0.5);
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

template <typename TL>
__global__ __launch_bounds__(THREADS) void sample_rows_kernel(const SampleArgs a) {
    __shared__ Shared s;
    const int row_at = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int V = a.V, segs = (V + SEG - 1) / SEG;
    const TL* const row = reinterpret_cast<const TL*>(a.logits + (int64_t)row_at * a.ld);
    double* const sums = reinterpret_cast<double*>(a.scratch) + (int64_t)row_at * segs;
    const RowAsks r = asks_of(a, row_at);

    float top = NEVER;
    int first = V;
    for (int g = wave; g < segs; g += NW) {
        Lane16<TL> x;
        x.load(row, V, g);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int i = g * SEG + x.at(e);
            if (x.v[e] > top || (x.v[e] == top && i < first)) top = x.v[e], first = i;
        }
    }
    const float mine = top;
    top = wave_max(top);
    if (lane == 0) s.fpart[wave] = top;
    __syncthreads();
    for (int w = 0; w < NW; w++) top = fmaxf(top, s.fpart[w]);
    if (threadIdx.x == 0) s.pick = V;
    __syncthreads();
    if (mine == top) atomicMin(&s.pick, first);
    __syncthreads();
    if (top == NEVER || r.greedy) {
        if (threadIdx.x == 0) a.ids[row_at] = top == NEVER ? -1 : s.pick;
        return;
    }
    const double scale = (double)(1ull << a.shift);
    Cut cut = {key_of(NEVER), V};
    if (r.top_k) cut = select(row, V, top, r.T, scale, cut, false, (uint32_t)r.k, 0ull, s);
    if (r.top_p) {
        unsigned long long m = 0;
        for (int g = wave; g < segs; g += NW) {
            Lane16<TL> x;
            x.load(row, V, g);
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (cut.holds(key_of(x.v[e]), g * SEG + x.at(e))) m += (unsigned long long)(weight_of(x.v[e], top, r.T) * scale + 0.5);
        }
        m = wave_sum(m);
        __syncthreads();
        if (lane == 0) s.mass[wave] = m;
        __syncthreads();
        m = 0;
        for (int w = 0; w < NW; w++) m += s.mass[w];
        cut = select(row, V, top, r.T, scale, cut, true, 0u, (unsigned long long)ceil(r.p * (double)m), s);
    }
    auto stays = [&](float l, int i) __attribute__((always_inline)) {
        if (l == NEVER || !cut.holds(key_of(l), i)) return 0.0;
        const double w = weight_of(l, top, r.T);
        return w < r.min_p && l != top ? 0.0 : w;
    };
    for (int g = wave; g < segs; g += NW) {
        Lane16<TL> x;
        x.load(row, V, g);
        double w = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) w += stays(x.v[e], g * SEG + x.at(e));
        w = wave_sum(w);
        if (lane == 0) sums[g] = w;
    }
    __syncthreads();
    // the segment: up to 1024 of them at a time
    double total = 0;
    for (int g0 = 0; g0 < segs; g0 += THREADS) {
        double all;
        scan_before(g0 + (int)threadIdx.x < segs ? sums[g0 + threadIdx.x] : 0.0, s.part, &all);
        total += all;
    }
    const double u = (double)a.u[row_at];
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

size_t sample_scratch_bytes(int B, int V) { return (((size_t)B * ((V + SEG - 1) / SEG) * 8) + 255) & ~(size_t)255; }

int launch_sample(const SampleArgs& a, int B, bool f32, hipStream_t st) {
    if (f32) hipLaunchKernelGGL(sample_rows_kernel<float>, dim3((unsigned)B), dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL(sample_rows_kernel<uint16_t>, dim3((unsigned)B), dim3(THREADS), 0, st, a);
    return check_hip(hipGetLastError(), "sample_rows_kernel launch");
}

}  // namespace mmx
