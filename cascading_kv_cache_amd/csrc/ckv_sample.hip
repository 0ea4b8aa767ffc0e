// A token a row, drawn from softmax(logits / temperature) cut off by top-k, top-p and min-p, with given random numbers.
//
//   Order: falling logits, equal ones by rising index.  x_i = (max - l_i) / T, w_i = exp(-x_i).
//   top-k keeps the first k, top-p what has less than p of their mass before it, min-p what has w_i >= min_p; the first one stays.
//   The token is the first whose running kept mass exceeds u times all of it.
//
// Every one of these sets is a beginning of the order, so nothing needs sorting but the elements around three borders: rows are laid into
// bins of x, 1/64 wide up to 32 (below that a weight is 2^-45 of the first one's: nothing), each with its count and mass; running sums say in
// which bins the borders lie, and the elements of those bins alone are collected and sorted.  Where they are too many to be (ties), the row is
// read again a byte of the order at a time.
//
// Masses are whole numbers, of 2^-44: sums are exact, whatever the order of the atomics that add them up, and a row means the same
// however many workgroups share it.  x is worked out in double (a logit of float32 less another has more digits than that, and a
// running sum over 10^5 tokens has as many borders that u may fall next to); of the exponential, 2^(-n/64) is a table in double and
// the rest, below 0.0055, a float32 polynomial: 2^-31 relative.
//
// A row is one workgroup's where there are rows enough to fill the chip, one launch with everything in LDS; fewer rows are shared out in
// slices over three launches (maximum; bins, and the last workgroup of a row to arrive finds the borders; elements, and the last one draws).
#include "ckv_common.h"

#include <algorithm>

namespace ckv {
namespace {

constexpr int kBins = 2048;
constexpr double kBinsPerUnit = 64.0, kFar = 32.0;   // kBins / kBinsPerUnit
constexpr int kListMax = 2048;                       // a power of two: the list is sorted in place
constexpr int kMaxSlices = 64;
constexpr int kMaxVocab = (1 << 20) - 1;             // of masses up to 2^44 each in 64 bits
constexpr uint64_t kOne = 1ull << 44;

// Which bins have to be looked at element by element, and what is known of the borders without that.
struct Borders {
    int from[3], to[3];   // top-k, top-p, the token; from > to: none
    int partial_k;        // the k-th element lies inside its bin
    int many;             // more elements in those bins than the list holds
    uint64_t mass_k;      // of the first k, unless partial
    uint64_t mass_min;    // of what min-p keeps
};

struct RowSpace {   // of a row that several workgroups share
    uint64_t mass[kBins + 1];
    uint32_t count[kBins + 1];
    uint32_t maxima[kMaxSlices];
    uint64_t mass_min;
    uint32_t arrived[2], listed;
    Borders borders;
    uint64_t list[kListMax];
};

struct SampleParams {
    const void* logits;
    int64_t stride;
    const float* uniforms;
    const float* temperature;   // a number a row, or null: the same for all
    const int64_t* top_k;
    const float* top_p;
    const float* min_p;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int64_t* tokens;
    float* logprobs;
    int vocab, slices;
    RowSpace* space;
};

struct Settings {
    double inv_t, far_min, p, u;   // far_min: the largest x that min-p keeps
    int k;
};

__device__ inline Settings settings_of(const SampleParams& s, int64_t row) {
    Settings r;
    const double t = s.temperature ? (double)s.temperature[row] : s.temperature_all;
    const int64_t k = s.top_k ? s.top_k[row] : s.top_k_all;
    r.k = k <= 0 || k > s.vocab ? s.vocab : (int)k;
    if (!(t > 0.0)) r.k = 1;   // the first one
    r.inv_t = t > 0.0 ? 1.0 / fmax(t, 1e-300) : 1.0;
    r.p = s.top_p ? (double)s.top_p[row] : s.top_p_all;
    const double least = s.min_p ? (double)s.min_p[row] : s.min_p_all;
    r.far_min = least > 0.0 ? (least < 1.0 ? -log(least) : 0.0) : 2 * kFar;
    r.u = (double)s.uniforms[row];
    return r;
}

// Rising with the value, zeros of either sign alike; NaN below everything.
__device__ inline uint32_t key_of(float l) {
    if (l != l) return 0;
    const uint32_t u = __float_as_uint(l + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr uint32_t kMinusInfinity = 0x007fffffu;

// x of a logit, or false: nothing of it counts
__device__ inline bool distance(float l, float m, double inv_t, double& x) {
    x = l == m ? 0.0 : ((double)m - (double)l) * inv_t;
    return x < kFar;
}
__device__ inline int bin_of(double x) { return (int)(x * kBinsPerUnit); }

__device__ inline void fill_table(double* table) {
    if (threadIdx.x < 64) table[threadIdx.x] = exp2(-(double)threadIdx.x / 64.0);
}

__device__ inline uint64_t mass_of(double x, const double* table) {
    const float n = rintf((float)x * 92.332482618935f);                     // 64 / ln 2
    const float r = (float)__builtin_fma(-(double)n, 0.010830424696249145, x);
    const float q = r * (-1.f + r * (0.5f + r * (-0.16666667f + r * 0.041666668f)));   // exp(-r) - 1
    const int i = (int)n;
    const double t = __longlong_as_double(__double_as_longlong(table[i & 63]) + (44 - (i >> 6)) * (1ll << 52));
    return (uint64_t)__double_as_longlong(__builtin_fma(t, (double)q, t) + 4503599627370496.0) & 0xfffffffffffffull;   // + 2^52: rounded to a whole number
}

// fn(index, value) for a slice of a row: vectors of 16 bytes between what lies in front of the first aligned one and behind the last.
template <typename T, typename Fn>
__device__ inline void for_each(const T* row, int vocab, int slice, int slices, Fn fn) {
    constexpr int kPer = 16 / (int)sizeof(T);
    struct alignas(16) Sixteen {
        T v[kPer];
    };
    const int head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    const int vectors = (vocab - head) / kPer, behind = head + vectors * kPer;
    if (slice == 0)
        for (int i = threadIdx.x; i < head; i += blockDim.x) fn(i, Elem<T>::to_float(row[i]));
    if (slice == slices - 1)
        for (int i = behind + threadIdx.x; i < vocab; i += blockDim.x) fn(i, Elem<T>::to_float(row[i]));
    const Sixteen* body = reinterpret_cast<const Sixteen*>(row + head);
    const int each = (vectors + slices - 1) / slices, end = min(vectors, (slice + 1) * each);
    constexpr int kAhead = 4;
    for (int i = slice * each + threadIdx.x; i < end; i += kAhead * blockDim.x) {
        Sixteen x[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++)
            if (i + a * (int)blockDim.x < end) x[a] = body[i + a * blockDim.x];
#pragma unroll
        for (int a = 0; a < kAhead; a++)
            if (i + a * (int)blockDim.x < end) {
#pragma unroll
                for (int e = 0; e < kPer; e++) fn(head + (i + a * (int)blockDim.x) * kPer + e, Elem<T>::to_float(x[a].v[e]));
            }
    }
}

// Running sums over the workgroup (any whole number of wavefronts): what lies in front of this thread; `all` gets the total.
template <typename V>
__device__ inline V before_me(V v, V* waves, V* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, many = blockDim.x >> 6;
    V s = v;
#pragma unroll
    for (int o = 1; o < CKV_WAVE; o <<= 1) {
        const V other = __shfl_up(s, o);
        if (lane >= o) s += other;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    V front = 0, total = 0;
    for (int w = 0; w < many; w++) {
        if (w < wave) front += waves[w];
        total += waves[w];
    }
    *all = total;
    return front + s - v;
}

__device__ inline uint32_t block_max(uint32_t v, uint32_t* waves) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); w++) v = max(v, waves[w]);
    return v;
}

struct Shared {
    uint64_t mass[kBins + 1];    // of a bin, then of all bins in front of it
    uint32_t count[kBins + 1];
    double table[64];
    uint64_t wide[16];
    uint32_t narrow[16];
    uint64_t mass_min;
    uint32_t listed, last;
    Borders borders;
    uint64_t answer[3];
};

struct Lists {
    uint64_t list[kListMax];     // order: (falling value, rising index)
    uint64_t running[kListMax];
};

// ---- the bins --------------------------------------------------------------------------------------------------------------------------

template <typename T>
__device__ inline void fill_bins(Shared& sh, const T* row, const SampleParams& s, const Settings& set, float m, int slice) {
    for (int i = threadIdx.x; i <= kBins; i += blockDim.x) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
    if (threadIdx.x == 0) sh.mass_min = 0;
    fill_table(sh.table);
    __syncthreads();
    uint64_t kept = 0;
    for_each(row, s.vocab, slice, s.slices, [&](int, float l) {
        double x;
        if (!distance(l, m, set.inv_t, x)) return;
        const uint64_t q = mass_of(x, sh.table);
        const int b = bin_of(x);
        atomicAdd((unsigned long long*)&sh.mass[b], (unsigned long long)q);
        atomicAdd(&sh.count[b], 1u);
        if (x <= set.far_min) kept += q;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) kept += __shfl_xor(kept, o);
    if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long*)&sh.mass_min, (unsigned long long)kept);
    __syncthreads();
}

// The first bin at whose end `reached` holds, which it then does behind every later one; the last bin if nowhere.
template <typename Fn>
__device__ inline int first_bin(Shared& sh, Fn reached) {
    __syncthreads();
    if (threadIdx.x == 0) sh.last = kBins - 1;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += blockDim.x)
        if (reached(b + 1) && (b == 0 || !reached(b))) sh.last = b;
    __syncthreads();
    return sh.last;
}

// u times a mass, as a whole number below it
__device__ inline uint64_t draw_below(double u, uint64_t mass) {
    const double t = u * (double)mass;
    const uint64_t w = t > 0.0 ? (t < 1.8e19 ? (uint64_t)t : ~0ull) : 0;
    return w < mass ? w : mass - 1;
}

// Bins become running sums, and the borders are looked up in them.
__device__ inline void find_borders(Shared& sh, const Settings& set) {
    constexpr int kMost = 8;
    const int each = kBins / blockDim.x;   // 2 or 8
    uint64_t m[kMost], all_m;
    uint32_t c[kMost], all_c;
    uint64_t sm = 0;
    uint32_t sc = 0;
    for (int i = 0; i < each; i++) {
        m[i] = sh.mass[threadIdx.x * each + i];
        c[i] = sh.count[threadIdx.x * each + i];
        sm += m[i];
        sc += c[i];
    }
    uint64_t fm = before_me(sm, sh.wide, &all_m);
    uint32_t fc = before_me(sc, sh.narrow, &all_c);
    for (int i = 0; i < each; i++) {
        sh.mass[threadIdx.x * each + i] = fm;
        sh.count[threadIdx.x * each + i] = fc;
        fm += m[i];
        fc += c[i];
    }
    if (threadIdx.x == 0) {
        sh.mass[kBins] = all_m;
        sh.count[kBins] = all_c;
    }
    __syncthreads();
    Borders r;
    r.partial_k = 0;
    r.mass_min = sh.mass_min;
    r.from[0] = r.from[1] = 1;
    r.to[0] = r.to[1] = 0;
    uint64_t low = all_m, high = all_m;   // of what is kept
    if (set.k < (int)all_c) {
        const int b = first_bin(sh, [&](int e) { return sh.count[e] >= (uint32_t)set.k; });
        low = high = sh.mass[b + 1];
        if (sh.count[b + 1] != (uint32_t)set.k) {
            low = max(sh.mass[b], kOne);
            r.partial_k = 1;
            r.from[0] = r.to[0] = b;
        }
    }
    r.mass_k = high;
    if (set.p < 1.0) {
        const double t0 = set.p * (double)low, t1 = set.p * (double)high;
        r.from[1] = first_bin(sh, [&](int e) { return (double)sh.mass[e] >= t0; });
        r.to[1] = first_bin(sh, [&](int e) { return (double)sh.mass[e] >= t1; });
        low = min(low, max(sh.mass[r.from[1]], kOne));
        high = min(high, sh.mass[r.to[1] + 1]);
    }
    low = min(low, r.mass_min);
    high = min(high, r.mass_min);
    const uint64_t d0 = draw_below(set.u, low), d1 = draw_below(set.u, high);
    r.from[2] = first_bin(sh, [&](int e) { return sh.mass[e] > d0; });
    r.to[2] = first_bin(sh, [&](int e) { return sh.mass[e] > d1; });
    uint32_t many = 0;
    for (int i = 0; i < 3; i++)
        if (r.from[i] <= r.to[i]) many += sh.count[r.to[i] + 1] - sh.count[r.from[i]];
    r.many = many > (uint32_t)kListMax;
    __syncthreads();
    if (threadIdx.x == 0) sh.borders = r;
    __syncthreads();
}

__device__ inline bool wanted(const Borders& r, int b) {
    return (b >= r.from[0] && b <= r.to[0]) || (b >= r.from[1] && b <= r.to[1]) || (b >= r.from[2] && b <= r.to[2]);
}

__device__ inline uint64_t order_of(float l, int i) { return ((uint64_t)~key_of(l) << 32) | (uint32_t)i; }
__device__ inline float logit_of(uint64_t order) { return value_of(~(uint32_t)(order >> 32)); }

// ---- the token -------------------------------------------------------------------------------------------------------------------------

__device__ inline void answer(const SampleParams& s, int64_t row, const Settings& set, float m, uint64_t order, uint64_t kept) {
    double x;
    distance(logit_of(order), m, set.inv_t, x);
    s.tokens[row] = (int64_t)(uint32_t)order;
    s.logprobs[row] = (float)(-x - log((double)kept * (1.0 / (double)kOne)));
}

// From the elements of the borders' bins, n of them.
__device__ inline void draw_from_list(Shared& sh, Lists& li, const SampleParams& s, int64_t row, const Settings& set, float m, int n) {
    const Borders r = sh.borders;
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += blockDim.x) li.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += blockDim.x) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const uint64_t va = li.list[a], vb = li.list[b];
                if ((va > vb) == ((a & k) == 0)) {
                    li.list[a] = vb;
                    li.list[b] = va;
                }
            }
            __syncthreads();
        }
    // Running mass up to and with each element; the bins between are added where the next one starts.
    const int each = (n + blockDim.x - 1) / blockDim.x, first = min(n, (int)threadIdx.x * each), end = min(n, first + each);
    auto bin_at = [&](int i) {
        double x;
        distance(logit_of(li.list[i]), m, set.inv_t, x);
        return bin_of(x);
    };
    uint64_t sum = 0, all;
    uint32_t rank = 0, all_rank;
    int prev = first > 0 && first < n ? bin_at(first - 1) : -1;
    const int prev0 = prev;
    auto step = [&](int i, uint64_t& mass, uint32_t& place) {
        double x;
        distance(logit_of(li.list[i]), m, set.inv_t, x);
        const int b = bin_of(x);
        if (b != prev) {
            mass += sh.mass[b] - sh.mass[prev + 1];
            place += sh.count[b] - sh.count[prev + 1];
            prev = b;
        }
        const uint64_t q = mass_of(x, sh.table);
        mass += q;
        place += 1;
        return q;
    };
    for (int i = first; i < end; i++) step(i, sum, rank);
    const uint64_t front = before_me(sum, sh.wide, &all);
    const uint32_t front_rank = before_me(rank, sh.narrow, &all_rank);
    if (threadIdx.x == 0) {
        sh.answer[0] = r.mass_k;
        sh.answer[1] = kOne;
        sh.answer[2] = (uint64_t)(n - 1);
    }
    __syncthreads();
    // top-k
    prev = prev0;
    uint64_t at = front;
    uint32_t place = front_rank;
    for (int i = first; i < end; i++) {
        step(i, at, place);
        li.running[i] = at;
        if (r.partial_k && place == (uint32_t)set.k) sh.answer[0] = at;
    }
    __syncthreads();
    uint64_t kept = sh.answer[0];
    if (set.p < 1.0) {   // the last one that has less than p of that before it
        const double t = set.p * (double)kept;
        prev = prev0;
        at = front;
        place = 0;
        for (int i = first; i < end; i++) {
            const uint64_t q = step(i, at, place);
            if ((double)(at - q) < t) atomicMax((unsigned long long*)&sh.answer[1], (unsigned long long)at);
        }
        __syncthreads();
        kept = min(kept, sh.answer[1]);
    }
    kept = min(kept, r.mass_min);
    const uint64_t d = draw_below(set.u, kept);
    for (int i = first; i < end; i++)
        if (li.running[i] > d && (i == 0 || li.running[i - 1] <= d)) sh.answer[2] = (uint64_t)i;
    __syncthreads();
    if (threadIdx.x == 0) answer(s, row, set, m, li.list[sh.answer[2]], kept);
}

// Without a list: the row is read once for every byte of the order.  In one bin, the first element at which `reached(count, mass)`, of all
// up to and with it, holds; returns the running mass there and the element.
template <typename T, typename Fn>
__device__ inline uint64_t search_row(Shared& sh, Lists& li, const T* row, const SampleParams& s, const Settings& set, float m, int bin, Fn reached,
                                      uint64_t& element) {
    uint64_t* masses = li.list;                                    // 256
    uint32_t* counts = reinterpret_cast<uint32_t*>(li.running);   // 256
    uint64_t prefix = 0, mass = sh.mass[bin];
    uint32_t count = sh.count[bin];
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += blockDim.x) {
            masses[i] = 0;
            counts[i] = 0;
        }
        __syncthreads();
        for_each(row, s.vocab, 0, 1, [&](int i, float l) {
            double x;
            if (!distance(l, m, set.inv_t, x) || bin_of(x) != bin) return;
            const uint64_t o = order_of(l, i);
            if (shift < 56 && (o >> (shift + 8)) != (prefix >> (shift + 8))) return;
            const int digit = (int)(o >> shift) & 255;
            atomicAdd((unsigned long long*)&masses[digit], (unsigned long long)mass_of(x, sh.table));
            atomicAdd(&counts[digit], 1u);
        });
        __syncthreads();
        // every thread walks over the 256 sums alike
        int digit = 0, last = 0;
        uint64_t last_mass = mass;
        uint32_t last_count = count;
        bool found = false;
        for (; digit < 256; digit++) {
            if (!counts[digit]) continue;
            last = digit;
            last_mass = mass;
            last_count = count;
            if (reached(count + counts[digit], mass + masses[digit])) {
                found = true;
                break;
            }
            mass += masses[digit];
            count += counts[digit];
        }
        if (!found) {   // rounding of a border at the bin's end: the last one
            digit = last;
            mass = last_mass;
            count = last_count;
        }
        prefix |= (uint64_t)digit << shift;
        if (shift == 0) mass += masses[digit];
    }
    element = prefix;
    __syncthreads();
    return mass;
}

template <typename T>
__device__ inline void draw_from_row(Shared& sh, Lists& li, const T* row_logits, const SampleParams& s, int64_t row, const Settings& set, float m) {
    const Borders r = sh.borders;
    uint64_t element, kept = r.mass_k;
    if (r.partial_k)
        kept = search_row(sh, li, row_logits, s, set, m, r.from[0], [&](uint32_t c, uint64_t) { return c >= (uint32_t)set.k; }, element);
    if (set.p < 1.0) {
        const double t = set.p * (double)kept;
        const int b = first_bin(sh, [&](int e) { return (double)sh.mass[e] >= t; });
        kept = min(kept, max(kOne, search_row(sh, li, row_logits, s, set, m, b, [&](uint32_t, uint64_t q) { return (double)q >= t; }, element)));
    }
    kept = min(kept, r.mass_min);
    const uint64_t d = draw_below(set.u, kept);
    const int b = first_bin(sh, [&](int e) { return sh.mass[e] > d; });
    search_row(sh, li, row_logits, s, set, m, b, [&](uint32_t, uint64_t q) { return q > d; }, element);
    if (threadIdx.x == 0) answer(s, row, set, m, element, kept);
}

__device__ inline void no_answer(const SampleParams& s, int64_t row) {   // no logit above minus infinity
    s.tokens[row] = -1;
    s.logprobs[row] = __uint_as_float(0x7fc00000u);
}

// ---- a workgroup a row -----------------------------------------------------------------------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(1024) sample_row_kernel(SampleParams s) {
    __shared__ Shared sh;
    __shared__ Lists li;
    const int64_t row = blockIdx.x;
    const T* logits = (const T*)s.logits + row * s.stride;
    const Settings set = settings_of(s, row);
    uint32_t top = 0;
    for_each(logits, s.vocab, 0, 1, [&](int, float l) { top = max(top, key_of(l)); });
    top = block_max(top, sh.narrow);
    if (top <= kMinusInfinity) {
        if (threadIdx.x == 0) no_answer(s, row);
        return;
    }
    const float m = value_of(top);
    fill_bins(sh, logits, s, set, m, 0);
    find_borders(sh, set);
    const Borders r = sh.borders;
    if (r.many) {
        draw_from_row(sh, li, logits, s, row, set, m);
        return;
    }
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    for_each(logits, s.vocab, 0, 1, [&](int i, float l) {
        double x;
        if (distance(l, m, set.inv_t, x) && wanted(r, bin_of(x))) li.list[atomicAdd(&sh.listed, 1u)] = order_of(l, i);
    });
    __syncthreads();
    draw_from_list(sh, li, s, row, set, m, (int)sh.listed);
}

// ---- several workgroups a row ----------------------------------------------------------------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(256) sample_max_kernel(SampleParams s) {
    __shared__ uint32_t waves[4];
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    for (int i = blockIdx.x * 256 + threadIdx.x; i <= kBins; i += gridDim.x * 256) {
        space.mass[i] = 0;
        space.count[i] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        space.mass_min = 0;
        space.arrived[0] = space.arrived[1] = space.listed = 0;
    }
    uint32_t top = 0;
    for_each((const T*)s.logits + row * s.stride, s.vocab, blockIdx.x, s.slices, [&](int, float l) { top = max(top, key_of(l)); });
    top = block_max(top, waves);
    if (threadIdx.x == 0) space.maxima[blockIdx.x] = top;
}

__device__ inline uint32_t top_of(const RowSpace& space, int slices) {
    uint32_t top = (int)(threadIdx.x & 63) < slices ? space.maxima[threadIdx.x & 63] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    return top;
}

// Is this the last of the row's workgroups to arrive?  Then what the others wrote before is there to be read.
__device__ inline bool last_to_arrive(uint32_t* arrived, int slices, uint32_t* shared) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *shared = atomicAdd(arrived, 1u) == (uint32_t)slices - 1;
    __syncthreads();
    if (!*shared) return false;
    __threadfence();
    return true;
}

template <typename V>
__device__ inline V read_through(const V* p) {   // past what this compute unit may hold of it
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T>
__global__ void __launch_bounds__(256) sample_bins_kernel(SampleParams s) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    const uint32_t top = top_of(space, s.slices);
    if (top <= kMinusInfinity) return;   // all of the row's workgroups
    const Settings set = settings_of(s, row);
    fill_bins(sh, (const T*)s.logits + row * s.stride, s, set, value_of(top), blockIdx.x);
    for (int b = threadIdx.x; b < kBins; b += 256)
        if (sh.count[b]) {
            atomicAdd((unsigned long long*)&space.mass[b], (unsigned long long)sh.mass[b]);
            atomicAdd(&space.count[b], sh.count[b]);
        }
    if (threadIdx.x == 0) atomicAdd((unsigned long long*)&space.mass_min, (unsigned long long)sh.mass_min);
    if (!last_to_arrive(&space.arrived[0], s.slices, &sh.last)) return;
    for (int b = threadIdx.x; b < kBins; b += 256) {
        sh.mass[b] = read_through(&space.mass[b]);
        sh.count[b] = read_through(&space.count[b]);
    }
    if (threadIdx.x == 0) sh.mass_min = read_through(&space.mass_min);
    __syncthreads();
    find_borders(sh, set);
    for (int b = threadIdx.x; b <= kBins; b += 256) {
        space.mass[b] = sh.mass[b];
        space.count[b] = sh.count[b];
    }
    if (threadIdx.x == 0) space.borders = sh.borders;
}

template <typename T>
__global__ void __launch_bounds__(256) sample_draw_kernel(SampleParams s) {
    __shared__ Shared sh;
    __shared__ Lists li;
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    const T* logits = (const T*)s.logits + row * s.stride;
    const uint32_t top = top_of(space, s.slices);
    if (top <= kMinusInfinity) {
        if (blockIdx.x == 0 && threadIdx.x == 0) no_answer(s, row);
        return;
    }
    const float m = value_of(top);
    const Settings set = settings_of(s, row);
    const Borders r = space.borders;
    if (!r.many)
        for_each(logits, s.vocab, blockIdx.x, s.slices, [&](int i, float l) {
            double x;
            if (distance(l, m, set.inv_t, x) && wanted(r, bin_of(x)))
                __hip_atomic_store(&space.list[atomicAdd(&space.listed, 1u)], order_of(l, i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        });
    if (!last_to_arrive(&space.arrived[1], s.slices, &sh.last)) return;
    for (int b = threadIdx.x; b <= kBins; b += 256) {
        sh.mass[b] = space.mass[b];
        sh.count[b] = space.count[b];
    }
    fill_table(sh.table);
    if (threadIdx.x == 0) sh.borders = r;
    __syncthreads();
    if (r.many) {
        draw_from_row(sh, li, logits, s, row, set, m);
        return;
    }
    const int n = (int)read_through(&space.listed);
    for (int i = threadIdx.x; i < n; i += 256) li.list[i] = read_through(&space.list[i]);
    __syncthreads();
    draw_from_list(sh, li, s, row, set, m, n);
}

// Slices of a row: four workgroups of four wavefronts to a compute unit over all rows, none with less than 2048 elements; one where the rows
// alone are as many as half of the compute units.
int slices_of(int64_t rows, int64_t vocab, int cus) {
    if (2 * rows >= cus) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kMaxSlices, 2 * cus / rows), vocab / 2048));
}

template <typename T>
int run_sample(const SampleParams& s, int64_t rows, hipStream_t stream) {
    if (s.slices == 1) {
        hipLaunchKernelGGL((sample_row_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, stream, s);
        CKV_HIP_TRY(hipGetLastError());
        return CKV_OK;
    }
    const dim3 grid(s.slices, (unsigned)rows);
    hipLaunchKernelGGL((sample_max_kernel<T>), grid, dim3(256), 0, stream, s);
    CKV_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((sample_bins_kernel<T>), grid, dim3(256), 0, stream, s);
    CKV_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((sample_draw_kernel<T>), grid, dim3(256), 0, stream, s);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

}  // namespace
}  // namespace ckv

extern "C" int64_t ckv_sample_workspace_bytes(int64_t rows, int64_t vocab) {
    using namespace ckv;
    DeviceInfo di;
    if (rows <= 0 || vocab <= 0 || vocab > kMaxVocab || current_device_info(&di)) return 0;
    return slices_of(rows, vocab, di.cus) > 1 ? rows * (int64_t)sizeof(RowSpace) : 0;
}

extern "C" int ckv_sample(const ckv_sample_args* a, void* stream_) {
    using namespace ckv;
    if (!a) return CKV_ERR_NULL;
    if (a->dtype != CKV_F32 && a->dtype != CKV_F16 && a->dtype != CKV_BF16) return CKV_ERR_DTYPE;
    if (a->rows < 0 || a->vocab <= 0 || (a->rows > 1 && a->logit_stride < 0)) return CKV_ERR_SHAPE;
    if (a->vocab > kMaxVocab || a->rows > 0x7fffffff) return CKV_ERR_UNSUPPORTED;
    if (a->rows == 0) return CKV_OK;
    if (!a->logits || !a->uniforms || !a->tokens || !a->logprobs) return CKV_ERR_NULL;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    SampleParams s;
    s.logits = a->logits;
    s.stride = a->logit_stride;
    s.uniforms = a->uniforms;
    s.temperature = a->temperatures;
    s.top_k = a->top_ks;
    s.top_p = a->top_ps;
    s.min_p = a->min_ps;
    s.temperature_all = a->temperature;
    s.top_k_all = a->top_k;
    s.top_p_all = a->top_p;
    s.min_p_all = a->min_p;
    s.tokens = a->tokens;
    s.logprobs = a->logprobs;
    s.vocab = (int)a->vocab;
    s.slices = slices_of(a->rows, a->vocab, di.cus);
    s.space = nullptr;
    if (s.slices > 1) {
        if (!a->workspace || a->workspace_bytes < a->rows * (int64_t)sizeof(RowSpace)) return CKV_ERR_WORKSPACE;
        if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return CKV_ERR_STRIDE;
        s.space = (RowSpace*)a->workspace;
    }
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    switch (a->dtype) {
        case CKV_F32: return run_sample<float>(s, a->rows, stream);
        case CKV_F16: return run_sample<__half>(s, a->rows, stream);
        default: return run_sample<__hip_bfloat16>(s, a->rows, stream);
    }
}
