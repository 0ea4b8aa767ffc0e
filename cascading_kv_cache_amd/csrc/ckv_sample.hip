// A token a row, drawn from softmax(logits / temperature) cut off by top-k, top-p and min-p, with given random numbers.
//
//   Order: falling logits, equal ones by rising index.  x_i = (max - l_i) / T, w_i = exp(-x_i).
//   top-k keeps the first k, top-p what has less than p of their mass before it, min-p what has w_i >= min_p; the first one stays.
//   The token is the first whose running kept mass exceeds u times all of it.
//
// Every one of these sets is a beginning of the order, so nothing needs sorting but the elements around four borders: rows are laid into
// bins of x, ln 2 / 64 wide up to 32 (a weight of 2^-46: what lies further is nothing), running sums say in which bins the borders lie, and
// the elements of those bins alone are collected and sorted.  Where they are too many to be (ties), the row is read again a byte of the order
// at a time.
//
// A weight is 2^(-n / 64), its bin's, times 1 + q, which is no more than 0.0055 from one: a bin adds up q in whole numbers of 2^-31 and counts,
// both in one 64-bit atomic, so that sums are exact whatever the order of the atomics.  Masses of bins, or of beginnings of one, are rounded to
// whole numbers of 2^-44: running sums over bins and over elements agree to the last digit (in double, an empty bin between two threads' sums
// had a mass of 10^-16).  x is worked out in double (a logit of float32 less another has more digits than that, and a running sum over 10^5
// tokens has as many borders that u may fall next to); q is a float32 polynomial: 2^-31 relative to the weight.
//
// A row is one workgroup's where it is short or there are rows enough to fill the chip, one launch with everything in LDS; long rows of which there
// are fewer are shared out in slices over three launches (maximum; bins, and the last workgroup of a row to arrive finds the borders; elements, and the
// last one draws).  256 rows of 128256 bfloat16 logits, the whole distribution: 71 us, about 10 of them the maximum (6.5 TB/s, the only time that they
// come from memory) and 25 the bins, which the vector ALU bounds, some thirty instructions an element.  One row, top-k 50 and top-p 0.95: 27 us
// (3.4, 12.4 and 11.6), chains of trips to memory and of barriers, 4.5 of it the borders.
#include "ckv_common.h"

#include <algorithm>

namespace ckv {
namespace {

constexpr double kFar = 32.0;
constexpr float kBinsPerUnit = 92.332482618935f;     // 64 / ln 2
constexpr double kBinWidth = 0.010830424696249145;
constexpr int kBins = 2956;                          // kFar of them, the last rounded up
constexpr int kListMax = 2048;                       // a power of two: the list is sorted in place
constexpr int kMaxSlices = 64;
constexpr int kThreads = 1024;
constexpr int kMaxVocab = (1 << 19) - 1;             // of numbers below 2^25 in the lower 44 bits of a bin, and their count in the upper 20
constexpr int kCountShift = 44;
constexpr uint64_t kOne = 1ull << 44;                // the mass of the first token
constexpr uint32_t kBias = 1u << 24;                 // makes q's whole number positive

// Which bins have to be looked at element by element, and what is known of the borders without that.
struct Borders {
    int from[4], to[4];   // top-k, top-p, min-p, the token; from > to: none
    int partial_k;        // the k-th element lies inside its bin
    int many;             // more elements in those bins than the list holds
    uint64_t mass_k;      // of the first k, unless partial
};

struct RowSpace {   // of a row that several workgroups share
    unsigned long long bins[kBins];
    unsigned long long mass[kBins + 1];
    uint32_t count[kBins + 1];
    float maxima[kMaxSlices];
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
    double inv_t, far_min, p, u;   // far_min: the largest x that min-p keeps, above kFar: no limit
    int k;
};

__device__ inline Settings settings_of(const SampleParams& s, int64_t row) {
    // all loads first, of something where there is no array: one trip to memory instead of five
    const float u = s.uniforms[row], t_row = (s.temperature ? s.temperature : s.uniforms)[row], p_row = (s.top_p ? s.top_p : s.uniforms)[row],
                least_row = (s.min_p ? s.min_p : s.uniforms)[row];
    const int64_t k_row = s.top_k ? s.top_k[row] : s.top_k_all;
    Settings r;
    const double t = s.temperature ? (double)t_row : s.temperature_all;
    const int64_t k = k_row;
    r.k = k <= 0 || k > s.vocab ? s.vocab : (int)k;
    if (!(t > 0.0)) r.k = 1;   // the first one
    r.inv_t = t > 0.0 ? 1.0 / fmax(t, 1e-300) : 1.0;
    r.p = s.top_p ? (double)p_row : s.top_p_all;
    const double least = s.min_p ? (double)least_row : s.min_p_all;
    r.far_min = least > 0.0 ? (least < 1.0 ? -log(least) : 0.0) : 2 * kFar;
    r.u = (double)u;
    return r;
}

// Rising with the value, zeros of either sign alike.
__device__ inline uint32_t key_of(float l) {
    const uint32_t u = __float_as_uint(l + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// x of a logit, or false: nothing of it counts
__device__ inline bool distance(float l, float m, double inv_t, double& x) {
    x = l == m ? 0.0 : ((double)m - (double)l) * inv_t;
    return x < kFar;
}
__device__ inline float bin_of(double x) { return rintf((float)x * kBinsPerUnit); }   // a whole number; rises with x

__device__ inline void fill_table(double* table) {
    if (threadIdx.x < 64) table[threadIdx.x] = exp2(-(double)threadIdx.x / 64.0);
}
__device__ inline double bin_weight(int n, const double* table) { return __longlong_as_double(__double_as_longlong(table[n & 63]) - (int64_t)(n >> 6) * (1ll << 52)); }

// q of a weight in its bin, in whole numbers of 2^-31 and biased
__device__ inline uint32_t rest_of(double x, float n) {
    const float r = (float)__builtin_fma(-(double)n, kBinWidth, x);
    const float q = r * (-1.f + r * (0.5f + r * (-0.16666667f + r * 0.041666668f)));   // exp(-r) - 1
    return (uint32_t)((int)rintf(q * 2147483648.f) + (int)kBias);
}
// The mass of some weights of bin n: their count in the upper bits, the sum of their rests in the lower ones.
__device__ inline uint64_t mass_of(int n, uint64_t some, const double* table) {
    const int64_t count = (int64_t)(some >> kCountShift), rests = (int64_t)(some & ((1ull << kCountShift) - 1));
    return (uint64_t)rint(bin_weight(n, table) * (double)((count << 31) + rests - count * (int64_t)kBias) * 8192.0);   // 2^44 / 2^31
}

// A slice of a row: vectors of 16 bytes between what lies in front of the first aligned one and behind the last.
template <typename T>
struct Slice {
    static constexpr int kPer = 16 / (int)sizeof(T), kAhead = 4;
    struct alignas(16) Sixteen {
        T v[kPer];
    };
    const T* row;
    const Sixteen* body;
    int vocab, head, behind, first, end;
    bool has_head, has_rest;
    Sixteen x[kAhead];
    __device__ Slice(const T* row_, int vocab_, int slice, int slices) : row(row_), vocab(vocab_) {
        head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
        const int vectors = (vocab - head) / kPer, each = (vectors + slices - 1) / slices;
        behind = head + vectors * kPer;
        body = reinterpret_cast<const Sixteen*>(row + head);
        first = slice * each + threadIdx.x;
        end = min(vectors, (slice + 1) * each);
        has_head = slice == 0;
        has_rest = slice == slices - 1;
    }
    __device__ void load(int from) {
#pragma unroll
        for (int a = 0; a < kAhead; a++)
            if (from + a * (int)blockDim.x < end) x[a] = body[from + a * blockDim.x];
    }
    // fn(index, value) for all of it, the first vectors of which are loaded
    template <typename Fn>
    __device__ void each_loaded(Fn fn) {
        if (has_head)
            for (int i = threadIdx.x; i < head; i += blockDim.x) fn(i, Elem<T>::to_float(row[i]));
        if (has_rest)
            for (int i = behind + threadIdx.x; i < vocab; i += blockDim.x) fn(i, Elem<T>::to_float(row[i]));
        for (int i = first; i < end; i += kAhead * blockDim.x) {
            if (i != first) load(i);
#pragma unroll
            for (int a = 0; a < kAhead; a++)
                if (i + a * (int)blockDim.x < end) {
#pragma unroll
                    for (int e = 0; e < kPer; e++) fn(head + (i + a * (int)blockDim.x) * kPer + e, Elem<T>::to_float(x[a].v[e]));
                }
        }
    }
};

template <typename T, typename Fn>
__device__ inline void for_each(const T* row, int vocab, int slice, int slices, Fn fn) {
    Slice<T> part(row, vocab, slice, slices);
    part.load(part.first);
    part.each_loaded(fn);
}

// Running sums over the workgroup (up to sixteen wavefronts): what lies in front of this thread; `all` gets the total.
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
    V w = lane < many ? waves[lane] : 0;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const V other = __shfl_up(w, o);
        if (lane >= o) w += other;
    }
    *all = __shfl(w, 15);
    const V front = __shfl(w, (wave + 63) & 63);
    return (wave ? front : 0) + s - v;
}

// The largest of all in front of this thread; 0 if there is none.
__device__ inline uint32_t latest_before_me(uint32_t v, uint32_t* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, many = blockDim.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < CKV_WAVE; o <<= 1) {
        const uint32_t other = __shfl_up(s, o);
        if (lane >= o) s = max(s, other);
    }
    __syncthreads();
    if (lane == 63) waves[wave] = s;
    const uint32_t before = __shfl_up(s, 1);
    __syncthreads();
    uint32_t w = lane < min(wave, many) ? waves[lane] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) w = max(w, __shfl_xor(w, o));
    return lane ? max(w, before) : w;
}

__device__ inline float block_max(float v, float* waves) {   // of sixteen wavefronts
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[threadIdx.x & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

struct Shared {
    unsigned long long mass[kBins + 1];   // of all bins in front of one; first the bins themselves
    uint32_t count[kBins + 1];
    double table[64];
    uint64_t wide[16];
    uint32_t narrow[16];
    float tops[16];
    uint32_t listed, last;
    int first[5], counted[2];
    Borders borders;
    unsigned long long answer[3];
};

struct Lists {
    uint64_t list[kListMax];     // order: (falling value, rising index)
    uint64_t before[kListMax];   // counts and rests of all in front
};

// ---- the bins --------------------------------------------------------------------------------------------------------------------------

__device__ inline void clear_bins(Shared& sh) {
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) sh.mass[i] = 0;
    fill_table(sh.table);
}

template <typename T>
__device__ inline void fill_bins(Shared& sh, Slice<T>& part, const Settings& set, float m) {
    __syncthreads();
    part.each_loaded([&](int, float l) {
        double x;
        if (!distance(l, m, set.inv_t, x)) return;
        const float n = bin_of(x);
        atomicAdd(&sh.mass[(int)n], (1ull << kCountShift) | rest_of(x, n));
    });
    __syncthreads();
}

// The first bin at whose end `reached` holds, which it then does behind every later one; the last bin if nowhere.
template <typename Fn>
__device__ inline int first_bin(Shared& sh, Fn reached) {
    __syncthreads();
    if (threadIdx.x == 0) sh.first[0] = kBins - 1;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += blockDim.x)
        if (reached(b + 1) && (b == 0 || !reached(b))) sh.first[0] = b;
    __syncthreads();
    return sh.first[0];
}

// u times a mass, as a whole number below it
__device__ inline uint64_t draw_below(double u, uint64_t mass) {
    const double t = u * (double)mass;
    const uint64_t w = t > 0.0 ? (t < 1.8e19 ? (uint64_t)t : ~0ull) : 0;
    return w < mass ? w : mass - 1;
}

// Bins become running sums, and the borders are looked up by the threads that have them: in registers, one exchange for top-k, one for top-p, one
// for the token.
__device__ inline void find_borders(Shared& sh, const Settings& set) {
    constexpr int kEach = (kBins + kThreads - 1) / kThreads;
    uint64_t m[kEach + 1], sm = 0, all_m;
    uint32_t c[kEach + 1], sc = 0, all_c;
    const int first = threadIdx.x * kEach;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const uint64_t b = first + i < kBins ? sh.mass[first + i] : 0;
        m[i] = first + i < kBins ? mass_of(first + i, b, sh.table) : 0;
        c[i] = (uint32_t)(b >> kCountShift);
        sm += m[i];
        sc += c[i];
    }
    if (threadIdx.x < 5) sh.first[threadIdx.x] = kBins - 1;
    uint64_t fm = before_me(sm, sh.wide, &all_m);   // its barriers let everybody read the bins first
    uint32_t fc = before_me(sc, sh.narrow, &all_c);
#pragma unroll
    for (int i = 0; i <= kEach; i++) {
        const uint64_t dm = i < kEach ? m[i] : 0;
        const uint32_t dc = i < kEach ? c[i] : 0;
        m[i] = fm;
        c[i] = fc;
        if (i < kEach && first + i < kBins) {
            sh.mass[first + i] = fm;
            sh.count[first + i] = fc;
        }
        fm += dm;
        fc += dc;
    }
    if (threadIdx.x == 0) {
        sh.mass[kBins] = all_m;
        sh.count[kBins] = all_c;
    }
    // the first bin at whose end `reached` holds, which it then does behind every later one; the last bin if nowhere
    auto look = [&](int slot, auto reached) {
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (first + i < kBins && reached(m[i + 1], c[i + 1]) && (first + i == 0 || !reached(m[i], c[i]))) sh.first[slot] = first + i;
    };
    Borders r;
    r.partial_k = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r.from[i] = 1;
        r.to[i] = 0;
    }
    uint64_t low = all_m, high = all_m;   // of what is kept
    const bool some = set.k < (int)all_c;
    if (some) look(0, [&](uint64_t, uint32_t e) { return e >= (uint32_t)set.k; });
    __syncthreads();
    if (some) {
        const int b = sh.first[0];
        low = high = sh.mass[b + 1];
        if (sh.count[b + 1] != (uint32_t)set.k) {
            low = max((uint64_t)sh.mass[b], kOne);
            r.partial_k = 1;
            r.from[0] = r.to[0] = b;
        }
    }
    r.mass_k = high;
    if (set.p < 1.0) {
        const double t0 = set.p * (double)low, t1 = set.p * (double)high;
        look(1, [&](uint64_t e, uint32_t) { return (double)e >= t0; });
        look(2, [&](uint64_t e, uint32_t) { return (double)e >= t1; });
        __syncthreads();
        r.from[1] = sh.first[1];
        r.to[1] = sh.first[2];
        low = min(low, max((uint64_t)sh.mass[r.from[1]], kOne));
        high = min(high, (uint64_t)sh.mass[r.to[1] + 1]);
    }
    if (set.far_min < kFar) {
        const int b = (int)bin_of(set.far_min);
        r.from[2] = r.to[2] = b;
        low = min(low, max((uint64_t)sh.mass[b], kOne));
        high = min(high, (uint64_t)sh.mass[b + 1]);
    }
    const uint64_t d0 = draw_below(set.u, low), d1 = draw_below(set.u, high);
    look(3, [&](uint64_t e, uint32_t) { return e > d0; });
    look(4, [&](uint64_t e, uint32_t) { return e > d1; });
    __syncthreads();
    r.from[3] = sh.first[3];
    r.to[3] = sh.first[4];
    uint32_t many = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (r.from[i] <= r.to[i]) many += sh.count[r.to[i] + 1] - sh.count[r.from[i]];
    r.many = many > (uint32_t)kListMax;
    if (threadIdx.x == 0) sh.borders = r;
    __syncthreads();
}

__device__ inline bool wanted(const Borders& r, int b) {
    return (b >= r.from[0] && b <= r.to[0]) || (b >= r.from[1] && b <= r.to[1]) || (b >= r.from[2] && b <= r.to[2]) || (b >= r.from[3] && b <= r.to[3]);
}

__device__ inline uint64_t order_of(float l, int i) { return ((uint64_t)~key_of(l) << 32) | (uint32_t)i; }
__device__ inline float logit_of(uint64_t order) { return value_of(~(uint32_t)(order >> 32)); }

// The elements of the borders' bins.  All of them lie in one stretch of values: two comparisons pass most of a row over.
template <typename T, typename Fn>
__device__ inline void for_wanted(Slice<T>& part, const Settings& set, float m, const Borders& r, Fn fn) {
    int low = kBins, high = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (r.from[i] <= r.to[i]) {
            low = min(low, r.from[i]);
            high = max(high, r.to[i]);
        }
    // a bin further on either side, and rounded outwards twice over
    const double least = (double)m - (high + 1.5) * kBinWidth / set.inv_t, most = (double)m - (low - 1.5) * kBinWidth / set.inv_t;
    const float floor = least > -3.4e38 ? (float)least - fabsf((float)least) * 2.4e-7f : -__builtin_huge_valf();
    const float ceiling = most < 3.4e38 ? (float)most + fabsf((float)most) * 2.4e-7f : __builtin_huge_valf();
    part.each_loaded([&](int i, float l) {
        if (l < floor || l > ceiling) return;
        double x;
        if (distance(l, m, set.inv_t, x) && wanted(r, (int)bin_of(x))) fn(order_of(l, i));
    });
}

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
    if (n <= kThreads / 2) {   // an element's place is the number of smaller ones, counted by as many threads as there are for each
        int log = 1;
        while (log < 6 && (n << (log + 1)) <= kThreads) log++;
        const int element = threadIdx.x >> log, part = threadIdx.x & ((1 << log) - 1);
        const uint64_t mine = element < n ? li.list[element] : 0;
        int place = 0;
        if ((int)((threadIdx.x & ~63u) >> log) < n)
            for (int i = part; i < n; i += 1 << log) place += li.list[i] < mine;
        for (int o = (1 << log) >> 1; o > 0; o >>= 1) place += __shfl_xor(place, o);
        __syncthreads();
        if (element < n && part == 0) li.list[place] = mine;
        __syncthreads();
    } else {
        // A thread compares one pair a step, a wavefront those of 128 neighbours: steps within them need no other wavefront.
        int size = kThreads;
        while (size < n) size <<= 1;
        for (int i = n + threadIdx.x; i < size; i += kThreads) li.list[i] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                if (j >= 2 * CKV_WAVE) __syncthreads();
                if ((int)threadIdx.x < size / 2) {
                    const int i = threadIdx.x, a = 2 * i - (i & (j - 1)), b = a + j;
                    const uint64_t va = li.list[a], vb = li.list[b];
                    if ((va > vb) == ((a & k) == 0)) {
                        li.list[a] = vb;
                        li.list[b] = va;
                    }
                }
                if (j >= 2 * CKV_WAVE) __syncthreads();
                else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        __syncthreads();
    }
    // A thread has two neighbours at most.  The running mass up to an element is that of the bins in front of its own and of the beginning of its
    // bin up to it: the weights between, counts and rests, are added up over the list, and the element where the bin begins is looked up.
    static_assert(kListMax <= 2 * kThreads, "two a thread");
    const int each = n > (int)blockDim.x ? 2 : 1, first = threadIdx.x * each;
    double x[2] = {};
    uint64_t some[2] = {}, run[2] = {};
    int bin[2] = {-1, -1};
    uint32_t begin[2] = {};   // of its bin, 1-based, in this thread
    int before = -1;
    if (first > 0 && first < n) {
        double xb;
        distance(logit_of(li.list[first - 1]), m, set.inv_t, xb);
        before = (int)bin_of(xb);
    }
    uint32_t latest = 0;
    for (int e = 0; e < each; e++)
        if (first + e < n) {
            distance(logit_of(li.list[first + e]), m, set.inv_t, x[e]);
            const float b = bin_of(x[e]);
            bin[e] = (int)b;
            some[e] = (1ull << kCountShift) | rest_of(x[e], b);
            if (bin[e] != before) latest = first + e + 1;
            before = bin[e];
            begin[e] = latest;
        }
    uint64_t all;
    uint64_t front = before_me(some[0] + some[1], sh.wide, &all);
    const uint32_t begun = latest_before_me(latest, sh.narrow);
    for (int e = 0; e < each; e++)
        if (first + e < n) {
            li.before[first + e] = front;
            front += some[e];
        }
    if (threadIdx.x == 0) {
        sh.answer[0] = r.mass_k;
        sh.answer[1] = sh.answer[2] = kOne;
        sh.counted[0] = sh.counted[1] = 0;
        sh.listed = 0;
    }
    __syncthreads();
    // How many of the list, which are its first ones: top-p and min-p keep beginnings of it.
    auto count = [&](int which, bool a, bool b) {
        const int many = __popcll(__ballot(a)) + __popcll(__ballot(b));
        if ((threadIdx.x & 63) == 0 && many) atomicAdd(&sh.counted[which], many);
    };
    const bool there[2] = {first < n, each == 2 && first + 1 < n};
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (there[e]) {
            const uint32_t from = (begin[e] ? begin[e] : begun) - 1;
            const uint64_t in_front = li.before[first + e] - li.before[from];
            run[e] = sh.mass[bin[e]] + mass_of(bin[e], in_front + some[e], sh.table);
            some[e] = sh.mass[bin[e]] + mass_of(bin[e], in_front, sh.table);   // and before it
            if (r.partial_k && sh.count[bin[e]] + (first + e - from) + 1 == (uint32_t)set.k) sh.answer[0] = run[e];
        }
    if (set.far_min < kFar) count(0, there[0] && x[0] <= set.far_min, there[1] && x[1] <= set.far_min);
    __syncthreads();
    uint64_t kept = sh.answer[0];
    if (set.p < 1.0) {   // those that have less than p of that before them
        const double t = set.p * (double)kept;
        count(1, there[0] && (double)some[0] < t, there[1] && (double)some[1] < t);
    }
    if (set.p < 1.0 || set.far_min < kFar) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (there[e]) {
                if (first + e + 1 == sh.counted[1]) sh.answer[1] = run[e];
                if (first + e + 1 == sh.counted[0]) sh.answer[2] = run[e];
            }
        __syncthreads();
        if (set.p < 1.0) kept = min(kept, (uint64_t)sh.answer[1]);
        if (set.far_min < kFar) kept = min(kept, max((uint64_t)sh.answer[2], (uint64_t)sh.mass[r.from[2]]));
    }
    const uint64_t d = draw_below(set.u, kept);
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (there[e] && run[e] > d && some[e] <= d) sh.listed = first + e;
    __syncthreads();
    if (threadIdx.x == 0) answer(s, row, set, m, li.list[sh.listed], kept);
}

// Without a list: the row is read once for every byte of the order.  In one bin, the first element at which `reached(count, mass)`, of all
// up to and with it, holds; returns the running mass there and the element.
template <typename T, typename Fn>
__device__ inline uint64_t search_row(Shared& sh, Lists& li, const T* row, const SampleParams& s, const Settings& set, float m, int bin, Fn reached,
                                    uint64_t& element) {
    unsigned long long* digits = reinterpret_cast<unsigned long long*>(li.list);   // 256
    uint64_t prefix = 0, front = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += blockDim.x) digits[i] = 0;
        __syncthreads();
        for_each(row, s.vocab, 0, 1, [&](int i, float l) {
            double x;
            if (!distance(l, m, set.inv_t, x)) return;
            const float n = bin_of(x);
            if ((int)n != bin) return;
            const uint64_t o = order_of(l, i);
            if (shift < 56 && (o >> (shift + 8)) != (prefix >> (shift + 8))) return;
            atomicAdd(&digits[(int)(o >> shift) & 255], (1ull << kCountShift) | rest_of(x, n));
        });
        __syncthreads();
        // every thread walks over the 256 sums alike; if none reaches (rounding, at the bin's end), the last one that is there does
        int digit = 0;
        uint64_t some = front;
        for (int i = 0; i < 256; i++) {
            if (!digits[i]) continue;
            digit = i;
            front = some;
            some += digits[i];
            if (reached(sh.count[bin] + (uint32_t)(some >> kCountShift), sh.mass[bin] + mass_of(bin, some, sh.table))) break;
        }
        prefix |= (uint64_t)digit << shift;
        if (shift == 0) front = some;
    }
    element = prefix;
    __syncthreads();
    return sh.mass[bin] + mass_of(bin, front, sh.table);
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
    if (set.far_min < kFar) {   // what of its bin min-p keeps
        unsigned long long* sum = reinterpret_cast<unsigned long long*>(li.list);
        __syncthreads();
        if (threadIdx.x == 0) *sum = 0;
        __syncthreads();
        for_each(row_logits, s.vocab, 0, 1, [&](int, float l) {
            double x;
            if (!distance(l, m, set.inv_t, x) || x > set.far_min) return;
            const float n = bin_of(x);
            if ((int)n == r.from[2]) atomicAdd(sum, (1ull << kCountShift) | rest_of(x, n));
        });
        __syncthreads();
        kept = min(kept, max(kOne, sh.mass[r.from[2]] + mass_of(r.from[2], *sum, sh.table)));
    }
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
__global__ void __launch_bounds__(kThreads) sample_row_kernel(SampleParams s) {
    __shared__ Shared sh;
    __shared__ Lists li;
    const int64_t row = blockIdx.x;
    const T* logits = (const T*)s.logits + row * s.stride;
    const Settings set = settings_of(s, row);
    Slice<T> part(logits, s.vocab, 0, 1);
    part.load(part.first);
    clear_bins(sh);
    float m = -__builtin_huge_valf();
    part.each_loaded([&](int, float l) { m = fmaxf(m, l); });   // NaN is passed over
    part.load(part.first);
    m = block_max(m, sh.tops);
    if (!(m > -__builtin_huge_valf())) {
        if (threadIdx.x == 0) no_answer(s, row);
        return;
    }
    fill_bins(sh, part, set, m);
    part.load(part.first);
    find_borders(sh, set);
    const Borders r = sh.borders;
    if (r.many) {
        draw_from_row(sh, li, logits, s, row, set, m);
        return;
    }
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    for_wanted(part, set, m, r, [&](uint64_t o) { li.list[atomicAdd(&sh.listed, 1u)] = o; });
    __syncthreads();
    const int n = (int)sh.listed;
    __syncthreads();
    draw_from_list(sh, li, s, row, set, m, n);
}

// ---- several workgroups a row ----------------------------------------------------------------------------------------------------------

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_max_kernel(SampleParams s) {
    __shared__ float waves[kThreads / 64];
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < kBins; i += gridDim.x * kThreads) space.bins[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) space.arrived[0] = space.arrived[1] = space.listed = 0;
    float m = -__builtin_huge_valf();
    for_each((const T*)s.logits + row * s.stride, s.vocab, blockIdx.x, s.slices, [&](int, float l) { m = fmaxf(m, l); });
    m = block_max(m, waves);
    if (threadIdx.x == 0) space.maxima[blockIdx.x] = m;
}

__device__ inline float maximum_of(const RowSpace& space, int slices) {   // of a slice, a lane each
    return (int)(threadIdx.x & 63) < slices ? space.maxima[threadIdx.x & 63] : -__builtin_huge_valf();
}
__device__ inline float top_of(float m) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    return m;
}

// Is this the last of the row's workgroups to arrive?  Then what the others wrote before is there to be read.  Everything that goes from one to
// another is written by atomics of the device's scope and read by such loads, past the caches of an XCD, so their end is all there is to wait
// for: a fence would have every wavefront write back and invalidate the L2.  That end is what vmcnt counts, of the stores and atomics of every
// wavefront in front of the barrier, and what a release would wait for too; its write-back of the L2 is for plain stores, of which there are none here
// (with release and acquire on the one addition 33 x 152064 takes 50 us instead of 46).
__device__ inline bool last_to_arrive(uint32_t* arrived, int slices, uint32_t* shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) *shared = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)slices - 1;
    __syncthreads();
    return *shared;
}

template <typename V>
__device__ inline V read_through(const V* p) {   // past what this compute unit may hold of it
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_bins_kernel(SampleParams s) {
    __shared__ Shared sh;
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    // everything there is to wait for on the way before the first of it is needed
    const float maximum = maximum_of(space, s.slices);
    Slice<T> part((const T*)s.logits + row * s.stride, s.vocab, blockIdx.x, s.slices);
    part.load(part.first);
    const Settings set = settings_of(s, row);
    clear_bins(sh);
    const float m = top_of(maximum);
    if (!(m > -__builtin_huge_valf())) return;   // all of the row's workgroups
    fill_bins(sh, part, set, m);
    for (int b = threadIdx.x; b < kBins; b += kThreads)
        if (sh.mass[b]) (void)__hip_atomic_fetch_add(&space.bins[b], sh.mass[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!last_to_arrive(&space.arrived[0], s.slices, &sh.last)) return;
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.mass[b] = read_through(&space.bins[b]);
    __syncthreads();
    find_borders(sh, set);
    for (int b = threadIdx.x; b <= kBins; b += kThreads) {
        space.mass[b] = sh.mass[b];
        space.count[b] = sh.count[b];
    }
    if (threadIdx.x == 0) space.borders = sh.borders;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_draw_kernel(SampleParams s) {
    __shared__ Shared sh;
    __shared__ Lists li;
    const int64_t row = blockIdx.y;
    RowSpace& space = s.space[row];
    const T* logits = (const T*)s.logits + row * s.stride;
    const float maximum = maximum_of(space, s.slices);
    const Borders r = space.borders;
    Slice<T> part(logits, s.vocab, blockIdx.x, s.slices);
    part.load(part.first);
    const Settings set = settings_of(s, row);
    const float m = top_of(maximum);
    if (!(m > -__builtin_huge_valf())) {   // then there are no borders either
        if (blockIdx.x == 0 && threadIdx.x == 0) no_answer(s, row);
        return;
    }
    if (!r.many) {   // a slice's elements are collected here and take their place in the row's list together
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        for_wanted(part, set, m, r, [&](uint64_t o) { li.list[atomicAdd(&sh.listed, 1u)] = o; });
        __syncthreads();
        const uint32_t n = sh.listed;
        if (threadIdx.x == 0) sh.last = n ? __hip_atomic_fetch_add(&space.listed, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        __syncthreads();
        const uint32_t at = sh.last;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) __hip_atomic_store(&space.list[at + i], li.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!last_to_arrive(&space.arrived[1], s.slices, &sh.last)) return;
    const int n = r.many ? 0 : (int)read_through(&space.listed);
    for (int b = threadIdx.x; b <= kBins; b += kThreads) {
        sh.mass[b] = space.mass[b];
        sh.count[b] = space.count[b];
    }
    for (int i = threadIdx.x; i < n; i += kThreads) li.list[i] = read_through(&space.list[i]);
    fill_table(sh.table);
    if (threadIdx.x == 0) sh.borders = r;
    __syncthreads();
    if (r.many) {
        draw_from_row(sh, li, logits, s, row, set, m);
        return;
    }
    draw_from_list(sh, li, s, row, set, m, n);
}

// Slices of a row: one workgroup to a compute unit over all rows, none with less than 4096 elements, where what they spare is more than the two
// launches and the exchanges cost.  A workgroup goes through 4000 elements in a microsecond (0.25e-3 us each) behind 13 us for the rest; three launches
// take 24 us and a twentieth of one more a row.  bfloat16, top-k 50 and top-p 0.95, a row: 8191 tokens in one workgroup 15 us, 8192 in two slices
// 25; 128 rows of 128256 in one 45 us, 127 in two 47, 64 in four 36 (about 44 in one).
int slices_of(int64_t rows, int64_t vocab, int cus) {
    const int64_t slices = std::min<int64_t>(std::min<int64_t>(kMaxSlices, cus / rows), vocab / 4096);
    if (slices < 2 || 0.25e-3 * (double)(vocab - vocab / slices) <= 11.0 + 0.05 * (double)rows) return 1;
    return (int)slices;
}

template <typename T>
int run_sample(const SampleParams& s, int64_t rows, hipStream_t stream) {
    if (s.slices == 1) {
        hipLaunchKernelGGL((sample_row_kernel<T>), dim3((unsigned)rows), dim3(kThreads), 0, stream, s);
        CKV_HIP_TRY(hipGetLastError());
        return CKV_OK;
    }
    const dim3 grid(s.slices, (unsigned)rows);
    hipLaunchKernelGGL((sample_max_kernel<T>), grid, dim3(kThreads), 0, stream, s);
    CKV_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((sample_bins_kernel<T>), grid, dim3(kThreads), 0, stream, s);
    CKV_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((sample_draw_kernel<T>), grid, dim3(kThreads), 0, stream, s);
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
