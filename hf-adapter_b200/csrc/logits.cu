// What is done to a row of logits between the head and the next token.
//
// Rules (both kernels), in fp32, z the logit of token v, c how often v was generated, seen whether it occurs in the history at all:
//   seen: z > 0 ? z / repetition : z * repetition;  then  z - frequency * c - presence * (c > 0) + bias[v];  not allowed: -inf.
// Draw (pick_kernel, filter_kernel), z / temperature, m the row's largest value, e = exp(z - m):
//   top-k  keeps z >= the k-th largest (ties stay);
//   top-p  keeps, in descending order (of equal values the lowest index first), every token with less than p of the mass of the
//          top-k survivors before it; the first always;
//   min-p  keeps e >= min_p;
//   token  = argmax of e / noise over what is kept (noise: independent Exp(1) variates, which makes it a draw from the
//            renormalised distribution); temperature <= 0: argmax of z.  The lowest index wins a tie.
// A NaN is never drawn, +inf counts as the largest finite number, and a quotient beyond it as the finite number at that end (a row
// of the type's lowest value is a row of equal tokens, not an empty one); a row without any token gives -1.
//
// A history is counted in shared memory, a word a token of the slice that a CTA holds (bit 31: in the prompt; below: times
// generated): integer atomics, so the order does not matter.  Every sum that is not of integers runs in a fixed order, and
// masses that are added by atomics are 64-bit fixed point (2^-40): results repeat bit for bit.
#include <cooperative_groups.h>

#include <cstddef>

#include "umma.cuh"

namespace cg = cooperative_groups;

namespace rwkv7 {
namespace lg {
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 1024;           // of a histogram
constexpr float BIN_SCALE = 32.0f;   // first histogram: m - z in steps of 1/32, the last bin takes the rest
constexpr int LIST = 1024;           // tokens that the short way sorts
constexpr unsigned int FEW = 32;     // of which sorting costs next to nothing
constexpr float MASS_UNIT = 1099511627776.0f;  // 2^40
constexpr float FLOAT_MAX = 3.402823466e38f;

typedef unsigned long long u64;

struct Part {  // what a CTA found, relative to its own largest value
    double sum;
    float max, score, z;
    int top, index;
};
struct Cut {
    unsigned int key;  // values with down_key <= key are kept
    int index;         // of values with exactly this key only tokens below this one
    u64 mass;          // of what the key keeps (by count only)
    bool found;
};
struct Shared {
    Part part[MAX_CLUSTER];           // first CTA: of every CTA
    Part warp_part[WARPS];
    double sum_of[MAX_CLUSTER];
    u64 mass_of[4][2][MAX_CLUSTER];   // [list][of the tokens above the window, of those on the list]
    u64 warp_mass[WARPS];
    double warp_sum[WARPS];
    Cut cut;
    float max[MAX_CLUSTER], warp_max[WARPS], warp_est[WARPS];
    int top[MAX_CLUSTER], warp_top[WARPS];
    unsigned int warp_count[WARPS];
    // from here on only where there are filters
    unsigned int count[BINS];         // this CTA's histogram
    unsigned int owned[BINS];         // the cluster's, for the bins that this CTA owns (the others' places stay unused)
    unsigned int upto[BINS];          // the cluster's, summed from bin 0
    unsigned int list_n[4];           // first CTA: places given out on a list: top-k's, its second try, top-p's, its second try
    unsigned int list_base, list_at;
    int bin, reach, window_first, window_last;  // reach: the last bin up to which there are no more than FEW tokens
    union {
        u64 list[LIST];  // first CTA: down_key << 32 | token
        struct {         // the descent
            unsigned int count[BINS], all_count[BINS];
            u64 mass[BINS], all_mass[BINS];
            u64 above_of[2][MAX_CLUSTER];  // [count, mass] of what lies above the range
            unsigned int ties[MAX_CLUSTER];
            unsigned int above_count, bin_count;
            u64 above_mass, bin_mass;
            int index_cut;
        } w;
    };
};
static_assert(offsetof(Shared, owned) % 8 == 0, "its bins are read in pairs");
constexpr int PICK_SHARED = (offsetof(Shared, count) + 15) / 16 * 16, FILTER_SHARED = (sizeof(Shared) + 15) / 16 * 16;
}  // namespace lg

struct Row {  // the rules of one row
    const int32_t* allowed;
    const float* bias;
    float repetition, presence, frequency;
    bool history;
};

__device__ __forceinline__ float param(const float* p, float v, int64_t row) { return p ? p[row] : v; }

__device__ __forceinline__ Row row_rules(const rwkv7_logit_rules& r, int64_t row) {
    Row o;
    o.allowed = r.allowed ? r.allowed + row * r.allowed_ld : nullptr;
    o.bias = r.bias ? r.bias + row * r.bias_ld : nullptr;
    o.history = r.tokens != nullptr;
    o.repetition = param(r.repetition, r.repetition_value, row);
    o.presence = param(r.presence, r.presence_value, row);
    o.frequency = param(r.frequency, r.frequency_value, row);
    return o;
}

// word: the token's history; products and differences rounded one by one
__device__ __forceinline__ float penalise(const Row& r, float z, unsigned int word) {
    if (word) {
        z = z > 0.0f ? z / r.repetition : z * r.repetition;
        const unsigned int c = word & 0x7fffffffu;
        z = __fsub_rn(__fsub_rn(z, __fmul_rn(r.frequency, (float)c)), c ? r.presence : 0.0f);
    }
    return z;
}

// One vector of VEC tokens from v0 on, of which those inside [0, V) count (the others become -inf); words: their history.
template <typename T, int VEC, bool RULES>
__device__ __forceinline__ void load_vector(const T* in, int v0, int V, const Row& r, const unsigned int* words, float (&z)[VEC]) {
    if (v0 >= 0 && v0 + VEC <= V) {
        const uint4 raw = *reinterpret_cast<const uint4*>(in + v0);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[i] = to_f<T>(e[i]);
        if constexpr (RULES) {
            if (r.history) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) z[i] = penalise(r, z[i], words[i]);
            }
            if (r.bias) {
                const float* b = r.bias + v0;
                if ((reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
                    for (int h = 0; h < VEC; h += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(b + h);
                        z[h] = __fadd_rn(z[h], q.x), z[h + 1] = __fadd_rn(z[h + 1], q.y);
                        z[h + 2] = __fadd_rn(z[h + 2], q.z), z[h + 3] = __fadd_rn(z[h + 3], q.w);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) z[i] = __fadd_rn(z[i], b[i]);
                }
            }
            if (r.allowed) {
                const int at = v0 >> 5, sh = v0 & 31;
                unsigned int bits = (unsigned int)r.allowed[at] >> sh;
                if (sh > 32 - VEC) bits |= (unsigned int)r.allowed[at + 1] << (32 - sh);  // (the vector's last token is in the next word)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (!((bits >> i) & 1)) z[i] = -INFINITY;
            }
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < VEC; ++i) {
            const int v = v0 + i;
            float x = -INFINITY;
            if (v >= 0 && v < V) {
                x = to_f<T>(in[v]);
                if constexpr (RULES) {
                    if (r.history) x = penalise(r, x, words[i]);
                    if (r.bias) x = __fadd_rn(x, r.bias[v]);
                    if (r.allowed && !((r.allowed[v >> 5] >> (v & 31)) & 1)) x = -INFINITY;
                }
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (k == i) z[k] = x;  // (no indexed registers)
        }
    }
}

// counts the history's tokens in [first, first + n) into words[0, n), n a multiple of 4; ids outside the vocabulary fall outside every
// slice.  Four ids a thread are on their way while the words are cleared, and while the four before them are counted.
__device__ __forceinline__ void count_history(const rwkv7_logit_rules& r, int64_t row, int first, int n, unsigned int* words) {
    constexpr int AHEAD = 4;
    int len = r.lengths ? r.lengths[row] : r.history;
    len = len < r.history ? len : r.history;
    const int prompt = r.prompt_lengths ? r.prompt_lengths[row] : 0, T = blockDim.x;
    const auto* wide = static_cast<const int64_t*>(r.tokens) + row * r.tokens_ld;
    const auto* narrow = static_cast<const int32_t*>(r.tokens) + row * r.tokens_ld;
    int64_t id[AHEAD];
    const auto request = [&](int i0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * T;
            id[u] = i >= len ? -1 : r.tokens_i64 ? wide[i] : (int64_t)narrow[i];
        }
    };
    request(threadIdx.x);
    for (int i = threadIdx.x * 4; i < n; i += T * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < len; i0 += AHEAD * T) {
        int at[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t d = id[u] - first;
            at[u] = id[u] >= 0 && d >= 0 && d < n ? (int)d : -1;
        }
        request(i0 + AHEAD * T);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (at[u] >= 0) {
                if (i0 + u * T >= prompt) atomicAdd(&words[at[u]], 1u);
                else atomicOr(&words[at[u]], 0x80000000u);
            }
    }
    __syncthreads();
}

// ---------------------------------------------------------------- rules alone
// grid (slices, rows); a row of any alignment is walked in 16-byte vectors that begin up to 16 bytes before it.  A slice's history is
// counted by its own CTA, which reads the row's whole history for that (out of L2 after the first): no second launch, no counts in memory.
// Bound by the launch and the chain history -> counts -> logits for a row or two, by issued instructions for many: device us, 65536 tokens fp16,
// one row and 300 tokens of history 3.6, 64 rows, 4096 tokens, a bias and a mask 14.2 (19.7 MB in and out: 1.4 TB/s), 256 rows, 300 tokens
// 26.7 (67 MB: 2.5 TB/s).
template <typename T>
__global__ void __launch_bounds__(512) process_logits_kernel(const T* logits, int64_t ld, const rwkv7_logit_rules rules, T* out,
                                                             int64_t out_ld, int V, int slice) {
    extern __shared__ unsigned int words[];
    constexpr int VEC = 16 / sizeof(T);
    const int64_t row = blockIdx.y;
    const T* in = logits + row * ld;
    T* o = out + row * out_ld;
    const int mis = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);  // elements before the row in its first vector
    const bool vec_out = (reinterpret_cast<uintptr_t>(o) / sizeof(T)) % VEC == (uintptr_t)mis;
    const int first = blockIdx.x * slice - mis;  // token of the slice's first place (may lie before the row)
    grid_dependency_wait();
    grid_launch_dependents();
    const Row r = row_rules(rules, row);
    if (r.history) count_history(rules, row, first, slice, words);
    for (int j = threadIdx.x * VEC; j < slice; j += blockDim.x * VEC) {
        const int v0 = first + j;
        if (v0 >= V) break;
        float z[VEC];
        load_vector<T, VEC, true>(in, v0, V, r, words + j, z);
        alignas(16) T res[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) res[i] = from_f<T>(z[i]);
        if (vec_out && v0 >= 0 && v0 + VEC <= V) {
            *reinterpret_cast<uint4*>(o + v0) = *reinterpret_cast<const uint4*>(res);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (v0 + i >= 0 && v0 + i < V) o[v0 + i] = res[i];
        }
    }
}

// ---------------------------------------------------------------- the draw
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ int linear_bin(float m, float z) {
    const float d = (m - z) * lg::BIN_SCALE;
    return d < (float)(lg::BINS - 1) ? (int)d : lg::BINS - 1;
}
// ascending keys for descending values (finite, no -0)
__device__ __forceinline__ unsigned int down_key(float z) {
    const unsigned int b = __float_as_uint(z);
    return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k : ~(k | 0x80000000u)); }
__device__ __forceinline__ lg::u64 fixed_mass(float e) { return __float2ull_rn(e * lg::MASS_UNIT); }
__device__ __forceinline__ lg::u64 share_of(double share, double mass) {
    const double want = ceil(share * mass);
    return want < 1.0 ? 1ull : (lg::u64)want;
}

// A slice is walked in its own vectors of VEC places by the thread that loaded them; `f(place, z)` for every token that is there.
template <int VEC, typename F>
__device__ __forceinline__ void each_token(const float* zs, int slice, F f) {
    for (int j = threadIdx.x * VEC; j < slice; j += lg::THREADS * VEC) {
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
            const float4 q = *reinterpret_cast<const float4*>(zs + j + h);
            const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (z[i] != -INFINITY) f(j + h + i, z[i]);
        }
    }
}

// log of a sum that is at least 1
__device__ __forceinline__ float log_sum(double sum) { return log1pf((float)(sum - 1.0)); }

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ lg::u64 warp_add(lg::u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ void warp_best(float& v, int& i, float& z) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o), y = __shfl_xor_sync(0xffffffffu, z, o);
        const int j = __shfl_xor_sync(0xffffffffu, i, o);
        if (better(w, j, v, i)) v = w, i = j, z = y;
    }
}
// the same value over the block, in every thread; `at` holds a place a warp and is not in use
template <typename V> __device__ __forceinline__ V block_add(V v, V* at) {
    v = warp_add(v);
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    v = lane < lg::WARPS ? at[lane] : V(0);
    v = warp_add(v);
    __syncthreads();
    return v;
}
// block maximum (lowest index first), in every thread
__device__ __forceinline__ void block_max_index(float& v, int& i, lg::Shared& s) {
    float none = 0.0f;
    warp_best(v, i, none);
    if ((threadIdx.x & 31) == 0) s.warp_max[threadIdx.x >> 5] = v, s.warp_top[threadIdx.x >> 5] = i;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    v = s.warp_max[lane % lg::WARPS], i = s.warp_top[lane % lg::WARPS];
    warp_best(v, i, none);
}
// the CTA's sum and best score (all threads' values relative to one maximum); valid in warp 0
__device__ __forceinline__ lg::Part block_part(lg::Part x, lg::Shared& s) {
    x.sum = warp_add(x.sum);
    warp_best(x.score, x.index, x.z);
    if ((threadIdx.x & 31) == 0) s.warp_part[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x < 32) {
        x = s.warp_part[threadIdx.x % lg::WARPS];
        if (threadIdx.x >= lg::WARPS) x.sum = 0.0, x.score = -1.0f, x.index = 0x7fffffff;
        x.sum = warp_add(x.sum);
        warp_best(x.score, x.index, x.z);
    }
    return x;
}

// ------------------------------ the descent: any number of equal or neighbouring values at a cut
// The cluster's histogram of counts and masses over `bin_of(z)` into every CTA; with ABOVE also count and mass of what it puts at -1
// (other values outside 0 .. BINS - 1 are left out).  Equal bins of a whole warp are added up first: a row of one value would queue
// at one address.
template <bool ABOVE, typename F>
__device__ __forceinline__ void histogram(const float* zs, int slice, float m, lg::Shared& s, cg::cluster_group& cl, lg::u64& above_count,
                                          lg::u64& above_mass, F bin_of) {
    const int C = cl.num_blocks(), rank = cl.block_rank(), per = lg::BINS / C, lane = threadIdx.x & 31;
    for (int b = threadIdx.x; b < lg::BINS; b += lg::THREADS) s.w.count[b] = 0, s.w.mass[b] = 0;
    __syncthreads();
    lg::u64 n_above = 0, q_above = 0;
    for (int j0 = threadIdx.x - lane; j0 < slice; j0 += lg::THREADS) {
        const int j = j0 + lane;
        const float z = j < slice ? zs[j] : -INFINITY;
        int b = lg::BINS;
        lg::u64 q = 0;
        if (z != -INFINITY) {
            b = bin_of(z);
            if (b < lg::BINS) q = fixed_mass(expf(z - m));
            if (ABOVE && b < 0) ++n_above, q_above += q;
        }
        const bool in = b >= 0 && b < lg::BINS;
        const int most = __reduce_max_sync(0xffffffffu, in ? b : -1);
        if (most < 0) continue;
        const unsigned int who = __ballot_sync(0xffffffffu, in);
        if (__all_sync(0xffffffffu, !in || b == most)) {
            q = warp_add(in ? q : 0);
            if (lane == 0) atomicAdd(&s.w.count[most], (unsigned int)__popc(who)), atomicAdd(&s.w.mass[most], q);
        } else if (in) {
            atomicAdd(&s.w.count[b], 1u);
            atomicAdd(&s.w.mass[b], q);
        }
    }
    if (ABOVE) {
        n_above = block_add(n_above, s.warp_mass), q_above = block_add(q_above, s.warp_mass);
        if ((int)threadIdx.x < C) {
            lg::Shared* o = cl.map_shared_rank(&s, threadIdx.x);
            o->w.above_of[0][rank] = n_above, o->w.above_of[1][rank] = q_above;
        }
    }
    cl.sync();
    if (ABOVE) {
        above_count = above_mass = 0;
        for (int c = 0; c < C; ++c) above_count += s.w.above_of[0][c], above_mass += s.w.above_of[1][c];
    }
    for (int b = rank * per + threadIdx.x; b < (rank + 1) * per; b += lg::THREADS) {
        unsigned int n = 0;
        lg::u64 q = 0;
        for (int c = 0; c < C; ++c) {
            lg::Shared* o = cl.map_shared_rank(&s, c);
            n += o->w.count[b], q += o->w.mass[b];
        }
        for (int c = 0; c < C; ++c) {
            lg::Shared* o = cl.map_shared_rank(&s, c);
            o->w.all_count[b] = n, o->w.all_mass[b] = q;
        }
    }
    cl.sync();
}

// first bin at which count (or mass) above the range plus that of bins 0 .. b reaches the target; results in s.w (bin = -1: none)
__device__ __forceinline__ void find_crossing(lg::Shared& s, bool by_mass, lg::u64 target, unsigned int base_count, lg::u64 base_mass) {
    static_assert(lg::BINS == 2 * lg::THREADS, "two bins a thread");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = 2 * threadIdx.x;
    const unsigned int n0 = s.w.all_count[b], n1 = s.w.all_count[b + 1];
    const lg::u64 q0 = s.w.all_mass[b], q1 = s.w.all_mass[b + 1];
    unsigned int n = n0 + n1;
    lg::u64 q = q0 + q1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned int tn = __shfl_up_sync(0xffffffffu, n, o);
        const lg::u64 tq = __shfl_up_sync(0xffffffffu, q, o);
        if (lane >= o) n += tn, q += tq;
    }
    if (lane == 31) s.warp_count[warp] = n, s.warp_mass[warp] = q;
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
    unsigned int an = base_count + n - n0 - n1;  // before this thread's bins
    lg::u64 aq = base_mass + q - q0 - q1;
    for (int w = 0; w < warp; ++w) an += s.warp_count[w], aq += s.warp_mass[w];
    const bool before = (by_mass ? aq : (lg::u64)an) >= target, first = (by_mass ? aq + q0 : (lg::u64)(an + n0)) >= target;
    const bool second = (by_mass ? aq + q0 + q1 : (lg::u64)(an + n0 + n1)) >= target;
    if (!before && second) {
        s.bin = first ? b : b + 1;
        s.w.bin_count = first ? n0 : n1, s.w.bin_mass = first ? q0 : q1;
        s.w.above_count = first ? an : an + n0, s.w.above_mass = first ? aq : aq + q0;
    }
    __syncthreads();
}

// Equal values at the cut, of which `need` are kept, lowest index first: the first token of this slice that is not kept.
__device__ __forceinline__ int tie_cut(const float* zs, int slice, int first, unsigned int key, unsigned int need, lg::Shared& s,
                                       cg::cluster_group& cl) {
    const int per = (slice + lg::THREADS - 1) / lg::THREADS, j0 = threadIdx.x * per, j1 = min(j0 + per, slice);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned int mine = 0;
    for (int j = j0; j < j1; ++j) mine += zs[j] != -INFINITY && down_key(zs[j]) == key;
    unsigned int upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned int t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) s.warp_count[warp] = upto;
    if (threadIdx.x == 0) s.w.index_cut = 0x7fffffff;
    __syncthreads();
    unsigned int total = 0, at = upto - mine;
    for (int w = 0; w < lg::WARPS; ++w) {
        if (w < warp) at += s.warp_count[w];
        total += s.warp_count[w];
    }
    const int C = cl.num_blocks(), rank = cl.block_rank();
    if ((int)threadIdx.x < C) cl.map_shared_rank(&s, threadIdx.x)->w.ties[rank] = total;
    cl.sync();
    unsigned int ahead = 0;
    for (int c = 0; c < rank; ++c) ahead += s.w.ties[c];
    if (ahead >= need) return 0;  // an earlier slice has them all
    at += ahead;
    for (int j = j0; j < j1; ++j)
        if (zs[j] != -INFINITY && down_key(zs[j]) == key && at++ == need) s.w.index_cut = first + j;
    __syncthreads();
    return s.w.index_cut;
}

// The key at which the descending order reaches `target` tokens (or mass), looked for in bins r0 .. r1 of the first histogram, then,
// if it is not there, in all of them: BINS finer ones of equal width (values near zero have many keys, neighbours of any
// value few), then ranges of keys.  A range that is kept as a whole ends the search; its last key is the cut.
__device__ __noinline__ lg::Cut descend(const float* zs, int slice, int first, float m, lg::Shared& s, cg::cluster_group& cl, bool by_mass,
                                        lg::u64 target, int r0, int r1) {
    using lg::Cut;
    Cut cut{0xffffffffu, 0x7fffffff, 0, false};  // (by count: fewer tokens than k)
    lg::u64 base_count = 0, base_mass = 0;
    float start, scale;
    const auto fine = [&](float z) {
        const int b = linear_bin(m, z);
        if (b < r0) return -1;
        if (b > r1) return lg::BINS;
        const float t = ((m - z) - start) * scale;
        return t < (float)(lg::BINS - 1) ? max((int)t, 0) : lg::BINS - 1;
    };
    for (;; r0 = 0, r1 = lg::BINS - 1) {
        start = (float)r0 / lg::BIN_SCALE, scale = lg::BIN_SCALE * (float)lg::BINS / (float)(r1 - r0 + 1);
        histogram<true>(zs, slice, m, s, cl, base_count, base_mass, fine);
        find_crossing(s, by_mass, target, (unsigned int)base_count, base_mass);
        if (s.bin >= 0 || (r0 == 0 && r1 == lg::BINS - 1)) break;
        __syncthreads();
    }
    if (s.bin >= 0) {
        // the last key of fine bins up to b: they rise with the key
        const auto last = [&](int b) {
            unsigned int lo = down_key(m), hi = down_key(-lg::FLOAT_MAX);
            while (lo < hi) {
                const unsigned int mid = lo + (hi - lo + 1) / 2;
                if (fine(key_value(mid)) <= b) lo = mid;
                else hi = mid - 1;
            }
            return lo;
        };
        unsigned int lo = fine(m) == s.bin ? down_key(m) : last(s.bin - 1) + 1, hi = last(s.bin);
        for (int level = 0;; ++level) {  // (32 bits of key in steps of 10: four refinements at most)
            const unsigned int above_count = s.w.above_count, count = s.w.bin_count;
            const lg::u64 above_mass = s.w.above_mass, mass = s.w.bin_mass;
            cut = Cut{hi, 0x7fffffff, above_mass + mass, true};
            // a single token, or (by count) all of them: the range is kept as a whole
            if (count == 1 || lo == hi || (!by_mass && above_count + count == target) || level == 4) {
                if (by_mass && count > 1) {
                    const lg::u64 each = mass / count, need = (target - above_mass + each - 1) / each;
                    if (need < count) cut.index = tie_cut(zs, slice, first, hi, (unsigned int)need, s, cl);
                }
                break;
            }
            const int bits = 32 - __clz(hi - lo), shift = bits > 10 ? bits - 10 : 0;
            histogram<false>(zs, slice, m, s, cl, base_count, base_mass, [&](float z) {
                const unsigned int k = down_key(z);
                return k >= lo && k <= hi ? (int)((k - lo) >> shift) : lg::BINS;
            });
            find_crossing(s, by_mass, target, above_count, above_mass);
            if (s.bin < 0) break;
            lo += (unsigned int)s.bin << shift;
            const unsigned int end = lo + ((1u << shift) - 1);
            hi = end < hi ? end : hi;
        }
    }
    cl.sync();  // (the next list lies where the first CTA may still be reading)
    return cut;
}

// ------------------------------ a window of bins around the cut, sorted
// Where a cut lies: its bin is known (by count), or the estimate is in the middle of it, towards its first or its last token, or
// the bin holds too few tokens to tell.
enum Where { kAround = 0, kHere = 1, kBefore = 2, kAfter = 3 };
// Which bins go on the list of the first CTA, in s.window_first, s.window_last (first > last: not even the cut's bin fits).  From the
// first bin if no more than `room` tokens may be kept, and then two bins more where the cut is estimated, and (as sorting so few costs the same) as many as
// hold FEW: where tokens are few they are heavy, and a cut that is missed by one may be many bins away.  Else the cut's bin, with its neighbours where it may
// lie there: what lies above is weighed and raced in passing, not sorted.
__device__ __forceinline__ void place_window(lg::Shared& s, int bin, int where, bool exact, unsigned int room) {
    if (threadIdx.x == 0) {
        const int wide = exact ? bin : min(bin + 2, lg::BINS - 1);
        int first = 0, last = max(wide, exact ? 0 : s.reach);
        if (s.upto[wide] > room) {
            first = where == kAround ? max(bin - 2, 0) : where == kBefore ? max(bin - 1, 0) : bin;
            last = where == kAround ? wide : where == kAfter ? min(bin + 1, lg::BINS - 1) : bin;
            auto tokens = [&] { return s.upto[last] - (first ? s.upto[first - 1] : 0); };
            while (first <= last && tokens() > lg::LIST) {
                if (last > bin) --last;
                else ++first;
            }
        }
        s.window_first = first, s.window_last = last;
    }
    __syncthreads();
}
// The cut's bin (s.bin: 4 * bin + where) and the window.  The bin is known by count (k > 0), or
// estimated: a bin's mass is taken as its count times e of its middle (1.6 % off at most).  Few heavy tokens make most of that
// error, above the cut, so what the estimate of the whole row is off by (`all`: the row's mass) is taken as the error at the cut too (of 64 rows of
// normal logits 4 missed a window of five bins without this); `where` says which neighbours the rest may reach.  The exact masses decide later.
__device__ __forceinline__ void choose_window(lg::Shared& s, unsigned int k, float want, float all, unsigned int room) {
    static_assert(lg::BINS == 2 * lg::THREADS, "two bins a thread");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = 2 * threadIdx.x;
    if (threadIdx.x == 0) s.bin = 4 * (lg::BINS - 1) + kAround;
    __syncthreads();
    if (k) {
        const unsigned int before = b ? s.upto[b - 1] : 0;
        if (before < k && s.upto[b + 1] >= k) s.bin = 4 * (s.upto[b] >= k ? b : b + 1) + kHere;
    } else {
        const unsigned int n0 = s.upto[b] - (b ? s.upto[b - 1] : 0), n1 = s.upto[b + 1] - s.upto[b];
        const float middle = expf(-((float)b + 0.5f) / lg::BIN_SCALE), q0 = (float)n0 * middle;
        const float q1 = (float)n1 * middle * 0.969233234f;  // e^(-1/32)
        float q = q0 + q1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float t = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) q += t;
        }
        if (lane == 31) s.warp_est[warp] = q;
        __syncthreads();
        float total = 0.0f, upto = 0.0f;
        for (int w = 0; w < lg::WARPS; ++w) {
            if (w == warp) upto = total;
            total += s.warp_est[w];
        }
        want = fmaxf(want + (total - all), 1e-30f);
        // each thread's bins begin at the very number at which its neighbour's end, so that one of them has the crossing (where
        // rounding makes it two, the first, in every CTA)
        q += upto;
        const float left = __shfl_up_sync(0xffffffffu, q, 1), before = lane ? left : upto;
        if (before < want && q >= want) {
            // what is left of the estimate's error is some hundredths of a bin that holds tokens enough
            const bool one = before + q0 >= want;
            const float part = one ? (want - before) / q0 : (want - before - q0) / q1;
            const int where = (one ? n0 : n1) < 16 ? kAround : part < 0.2f ? kBefore : part > 0.8f ? kAfter : kHere;
            atomicMin(&s.bin, 4 * (one ? b : b + 1) + where);
        }
    }
    __syncthreads();
    place_window(s, s.bin >> 2, s.bin & 3, k != 0, room);
}

// list[0, n) ascending, n at most LIST; what pads it to a power of two is the largest key
__device__ __forceinline__ void sort_list(lg::u64* list, int n) {
    int size = 32;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += lg::THREADS) list[i] = ~0ull;
    __syncthreads();
    // a pair a thread, who meet without the others: one warp up to 64 tokens (50: 4600 -> 1300 cycles), a barrier of their own above
    const int t = threadIdx.x, threads = size / 2 < 32 ? 32 : size / 2;
    if (t < threads)
        for (int span = 2; span <= size; span *= 2)
            for (int d = span / 2; d > 0; d /= 2) {
                const int i = 2 * t - (t & (d - 1));
                if (t < size / 2) {
                    const lg::u64 a = list[i], b = list[i + d];
                    if ((a > b) == ((i & span) == 0)) list[i] = b, list[i + d] = a;
                }
                if (threads == 32) __syncwarp();
                else asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
            }
    __syncthreads();
}

// what the two places of this thread on the sorted list hold, and the mass before them
struct Places {
    float z[2], e[2];
    lg::u64 w[2], before, total;
};
__device__ __forceinline__ Places weigh_list(const lg::u64* list, int n, float m, lg::u64 above, lg::Shared& s) {
    static_assert(lg::LIST == 2 * lg::THREADS, "two places a thread");
    const int i0 = threadIdx.x * 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Places o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        o.z[i] = i0 + i < n ? key_value((unsigned int)(list[i0 + i] >> 32)) : -INFINITY;
        o.e[i] = expf(o.z[i] - m), o.w[i] = fixed_mass(o.e[i]);
    }
    lg::u64 upto = o.w[0] + o.w[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const lg::u64 t = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += t;
    }
    if (lane == 31) s.warp_mass[warp] = upto;
    __syncthreads();
    o.before = above + upto - o.w[0] - o.w[1], o.total = above;
    for (int w = 0; w < lg::WARPS; ++w) {
        const lg::u64 t = s.warp_mass[w];
        if (w < warp) o.before += t;
        o.total += t;
    }
    __syncthreads();
    return o;
}
// places of the sorted list that hold keys up to `key`
__device__ __forceinline__ int places_upto(const lg::u64* list, int n, unsigned int key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if ((unsigned int)(list[mid] >> 32) <= key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// e = exp(d) for the sums and races over all tokens: one ex2, off by 2^-22 and |d| 2^-23 (exactly 1 at 0); what decides a cut by
// mass uses expf
__device__ __forceinline__ float fast_exp(float d) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.44269504f));
    return e;
}
// e / q of a race, off by 2^-22: equal operands give equal scores, nearer ones are nearer than the noise is random
__device__ __forceinline__ float race_score(float e, float q) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(q));
    return e * r;
}

// The best score of what lies above the window (no e below `least`) in this CTA's slice, to the first CTA.  A function of its own: inlined
// it costs rows that do not need it half a microsecond of 16.
template <int VEC>
__device__ __noinline__ void race_above(int slice, int first, float m, float least, const float* q) {
    extern __shared__ __align__(16) unsigned char smem[];
    lg::Shared& s = *reinterpret_cast<lg::Shared*>(smem);
    const float* zs = reinterpret_cast<const float*>(smem + lg::FILTER_SHARED);
    cg::cluster_group cl = cg::this_cluster();
    const float edge = (float)s.window_first;  // linear_bin() below it
    lg::Part best{0.0, m, -1.0f, 0.0f, 0, 0x7fffffff};
    for (int j = threadIdx.x * VEC; j < slice; j += lg::THREADS * VEC) {
        float z[VEC], n[VEC];
        bool over[VEC], any = false;
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
            const float4 w = *reinterpret_cast<const float4*>(zs + j + h);
            z[h] = w.x, z[h + 1] = w.y, z[h + 2] = w.z, z[h + 3] = w.w;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) over[i] = (m - z[i]) * lg::BIN_SCALE < edge, any |= over[i];
        if (!any) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[i] = q[over[i] ? first + j + i : 0];  // (requested together, as in finish())
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float e = fast_exp(z[i] - m), score = race_score(e, n[i]);
            if (over[i] && e >= least && score > best.score) best.score = score, best.index = first + j + i, best.z = z[i];
        }
    }
    best = block_part(best, s);
    if (threadIdx.x == 0) cl.map_shared_rank(&s, 0)->part[cl.block_rank()] = best;
}

// Every token of the window, no key beyond `limit`, to the first CTA's list; the masses (if asked for) of it and of what lies
// above to every CTA.  `few`: so few tokens that each takes its own place, else a CTA takes places for all of its at once.  Ends
// with a cluster barrier.
template <int VEC>
__device__ __forceinline__ void gather(const float* zs, int slice, int first, float m, lg::Shared& s, cg::cluster_group& cl, int turn,
                                       unsigned int limit, bool masses, bool few) {
    using lg::u64;
    const int w0 = s.window_first, w1 = s.window_last, C = cl.num_blocks(), rank = cl.block_rank();
    lg::Shared* head = cl.map_shared_rank(&s, 0);
    u64 mine = 0;  // (tokens of the window in this slice; some may lie beyond the limit)
    if (!few) {
        for (int b = w0 + threadIdx.x; b <= w1; b += lg::THREADS) mine += s.count[b];
        mine = block_add(mine, s.warp_mass);
        if (threadIdx.x == 0) s.list_base = mine ? atomicAdd(&head->list_n[turn], (unsigned int)mine) : 0, s.list_at = 0;
        __syncthreads();
    }
    u64 above = 0, listed = 0;
    if (few || mine || (masses && w0))
        each_token<VEC>(zs, slice, [&](int j, float z) {
            const int b = linear_bin(m, z);
            if (b > w1) return;
            const u64 e = masses ? fixed_mass(expf(z - m)) : 0;
            if (b < w0) {
                above += e;
                return;
            }
            const unsigned int key = down_key(z);
            const bool in = key <= limit;
            if (in) listed += e;
            const unsigned int at = few ? atomicAdd(&head->list_n[turn], 1u) : s.list_base + atomicAdd(&s.list_at, 1u);
            head->list[at] = in ? (u64)key << 32 | (unsigned int)(first + j) : ~0ull;
        });
    if (masses) {
        if (w0) above = block_add(above, s.warp_mass);
        listed = block_add(listed, s.warp_mass);
        if ((int)threadIdx.x < C) {
            lg::Shared* o = cl.map_shared_rank(&s, threadIdx.x);
            o->mass_of[turn][0][rank] = above, o->mass_of[turn][1][rank] = listed;
        }
    }
    cl.sync();
}

// The draw of one row, and which of its filters are on
struct Draw {
    float temperature, p, min_p;
    int k;
    bool greedy, by_k, by_p;
};
__device__ __forceinline__ Draw row_draw(const rwkv7_draw_params& d, bool noise, int64_t row, int V) {
    Draw o;
    o.temperature = noise ? param(d.temperature, d.temperature_value, row) : 0.0f;
    o.greedy = !(o.temperature > 0.0f);
    o.k = d.top_k ? d.top_k[row] : d.top_k_value;
    o.p = param(d.top_p, d.top_p_value, row), o.min_p = param(d.min_p, d.min_p_value, row);
    o.by_k = !o.greedy && o.k > 0 && o.k < V, o.by_p = !o.greedy && o.p < 1.0f;
    return o;
}

// z / t for finite results below 1e37 as a product with 1 / t and one correction step (the correctly rounded quotient); the rest
// (what is masked, NaN, out of range) on its own
__device__ __forceinline__ float over_temperature(float x, float t, float inv) {
    const float q = x * inv;
    float z = fmaf(fmaf(-q, t, x), inv, q) + 0.0f;  // (-0 becomes 0)
    if (!(fabsf(q) < 1e37f)) z = x > -INFINITY ? fmaxf(fminf(x / t, lg::FLOAT_MAX), -lg::FLOAT_MAX) : -INFINITY;  // (NaN compares false)
    return z;
}

// This CTA's slice of a row, ruled and divided, to zs; its largest value with the first token that has it
template <typename T, bool RULES>
__device__ __forceinline__ void load_row(const T* in, int first, int V, int slice, const rwkv7_logit_rules& rules, int64_t row, const Draw& d,
                                         float* zs, float& m, int& top) {
    constexpr int VEC = 16 / sizeof(T);
    Row r{};
    if constexpr (RULES) {
        r = row_rules(rules, row);
        if (r.history) count_history(rules, row, first, slice, reinterpret_cast<unsigned int*>(zs));
    }
    const float t = d.greedy ? 1.0f : d.temperature, inv = __frcp_rn(t);
    m = -INFINITY, top = 0x7fffffff;
    for (int j = threadIdx.x * VEC; j < slice; j += lg::THREADS * VEC) {
        const int v0 = first + j;
        float z[VEC];
        load_vector<T, VEC, RULES>(in, v0, V, r, reinterpret_cast<unsigned int*>(zs) + j, z);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            z[i] = over_temperature(z[i], t, inv);
            if (z[i] > m) m = z[i], top = v0 + i;
        }
#pragma unroll
        for (int h = 0; h < VEC; h += 4) *reinterpret_cast<float4*>(zs + j + h) = make_float4(z[h], z[h + 1], z[h + 2], z[h + 3]);
    }
}

// The largest value of the row, in every CTA of the cluster.  Ends with a cluster barrier.
__device__ __forceinline__ void row_max(float& m, int& top, lg::Shared& s, cg::cluster_group& cl) {
    const int C = cl.num_blocks(), rank = cl.block_rank();
    if ((int)threadIdx.x < C) {
        lg::Shared* o = cl.map_shared_rank(&s, threadIdx.x);
        o->max[rank] = m, o->top[rank] = top;
    }
    cl.sync();
    m = s.max[0], top = s.top[0];
    for (int c = 1; c < C; ++c)
        if (better(s.max[c], s.top[c], m, top)) m = s.max[c], top = s.top[c];
}

// The row's answer from the parts of its CTAs (valid in thread 0)
__device__ __forceinline__ void answer(const lg::Part& mine, bool greedy, lg::Shared& s, cg::cluster_group& cl, long long* token, float* logprob) {
    using lg::Part;
    const int C = cl.num_blocks(), rank = cl.block_rank();
    if (threadIdx.x == 0) cl.map_shared_rank(&s, 0)->part[rank] = mine;
    cl.sync();
    if (rank == 0 && threadIdx.x < 32) {
        Part x = s.part[threadIdx.x % C];
        if ((int)threadIdx.x >= C) x = Part{0.0, -INFINITY, -1.0f, 0.0f, 0x7fffffff, 0x7fffffff};
        float most = x.max, none = 0.0f;
        int at = x.top;
        warp_best(most, at, none);
        const float f = x.max == -INFINITY ? 0.0f : expf(x.max - most);
        const double sum = warp_add(x.sum * (double)f);
        if (x.index != 0x7fffffff) x.score *= f;
        warp_best(x.score, x.index, x.z);
        if (threadIdx.x == 0) {
            // (noise of NaN alone: the most likely token)
            const bool empty = most == -INFINITY, drawn = !greedy && x.index != 0x7fffffff;
            *token = empty ? -1 : drawn ? x.index : at;
            if (logprob) *logprob = empty ? -INFINITY : ((drawn ? x.z : most) - most) - log_sum(sum);
        }
    }
}

// Sum of exponentials and the race over this CTA's tokens that `keep(key, token, e)` lets in, and the row's answer from the parts
template <int VEC, typename F>
__device__ __noinline__ void finish(int slice, int first, float m, int top, bool greedy, const float* q, long long* token, float* logprob, F keep) {
    using lg::Part;
    extern __shared__ __align__(16) unsigned char smem[];
    lg::Shared& s = *reinterpret_cast<lg::Shared*>(smem);
    const float* zs = reinterpret_cast<const float*>(smem + lg::FILTER_SHARED);
    cg::cluster_group cl = cg::this_cluster();
    const bool sums = logprob != nullptr;
    Part best{0.0, m, -1.0f, 0.0f, top, 0x7fffffff};
    int ones = 0;  // e = 1 is counted apart: a sure token's log-probability is all in the small terms
    if ((sums || !greedy) && m != -INFINITY)
        for (int j = threadIdx.x * VEC; j < slice; j += lg::THREADS * VEC) {
            float z[VEC], e[VEC], n[VEC];
            bool in[VEC];
#pragma unroll
            for (int h = 0; h < VEC; h += 4) {
                const float4 w = *reinterpret_cast<const float4*>(zs + j + h);
                z[h] = w.x, z[h + 1] = w.y, z[h + 2] = w.z, z[h + 3] = w.w;
            }
            bool any = false;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                e[i] = fast_exp(z[i] - m);  // (0 of what is not there)
                in[i] = !greedy && z[i] != -INFINITY && keep(z[i], first + j + i, e[i]);
                n[i] = 1.0f, any |= in[i];
            }
            // the noise of what is kept, requested together: no load waits for a condition (of the others the first token's is read instead).
            // 256 rows, top-k 5000: 152 -> 138 us, 64 rows 34.9 -> 36.8, one row 21.4 -> 20.8
            if (any) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) n[i] = q[in[i] ? first + j + i : 0];
            }
#pragma unroll
            for (int h = 0; h < VEC; h += 4) {
                float part = 0.0f;
#pragma unroll
                for (int i = h; i < h + 4; ++i) {
                    if (e[i] == 1.0f) ++ones;
                    else part += e[i];
                    const float score = race_score(e[i], n[i]);
                    if (in[i] && score > best.score) best.score = score, best.index = first + j + i, best.z = z[i];  // (tokens come in order)
                }
                best.sum += (double)part;
            }
        }
    best.sum += (double)ones;
    best = block_part(best, s);
    answer(best, greedy, s, cl, token, logprob);
}

// Rows without any filter: one pass over logits and noise, everything relative to the largest value that a thread has met so far.
// The cluster of a row meets once, at the end, to compare its parts.  Bound by the launch and that chain for few rows, by issued instructions (0.6 a
// cycle and scheduler, 35 a warp for its 32 tokens) for many.  Device us, 65536 tokens fp16, greedy / drawn: one row 4.3 / 5.4, 64 rows 6.6 / 10.0, 256 rows
// 19.1 / 29.4 (33.6 MB and 101 MB: 1.8 and 3.4 TB/s); fp32 logits, 256 rows 21.4 / 31.5 (4.3 TB/s).
template <typename T, bool RULES>
__global__ void __launch_bounds__(lg::THREADS, 2) pick_kernel(const T* __restrict__ logits, int64_t ld, const rwkv7_logit_rules rules,
                                                              const rwkv7_draw_params draw, const float* __restrict__ noise, int64_t noise_ld,
                                                              long long* __restrict__ token, float* __restrict__ logprob, int V, int slice) {
    using namespace lg;
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    unsigned int* words = reinterpret_cast<unsigned int*>(smem + PICK_SHARED);  // the slice's history, where there is one
    cg::cluster_group cl = cg::this_cluster();
    constexpr int VEC = 16 / sizeof(T);
    const int rank = cl.block_rank();
    const int64_t row = blockIdx.x / cl.num_blocks();
    const T* in = logits + row * ld;
    const int first = rank * slice - (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);
    cluster_arrive_relaxed();  // this CTA runs: the others may write into its shared memory
    grid_dependency_wait();
    grid_launch_dependents();
    const float temperature = noise ? param(draw.temperature, draw.temperature_value, row) : 0.0f;
    const bool greedy = !(temperature > 0.0f), sums = logprob != nullptr;
    const float t = greedy ? 1.0f : temperature, inv = __frcp_rn(t);
    const float* q = greedy ? nullptr : noise + row * noise_ld;
    const bool vectors = ((reinterpret_cast<uintptr_t>(q) / 4 + first) & 3) == 0;
    Row r{};
    if constexpr (RULES) {
        r = row_rules(rules, row);
        if (r.history) count_history(rules, row, first, slice, words);
    }
    Part x{0.0, -INFINITY, 0.0f, 0.0f, 0x7fffffff, 0x7fffffff};  // (a token's score is positive, that of a masked one 0)
    float small = 0.0f;
    int ones = 0;  // e = 1 is counted apart: a sure token's log-probability is all in the small terms
    constexpr int TOK = 8;  // tokens a turn
#pragma unroll 2
    for (int j = threadIdx.x * TOK; j < slice; j += THREADS * TOK) {
        const int v0 = first + j;
        if (v0 >= V) break;
        float z[TOK], n[TOK];
#pragma unroll
        for (int i = 0; i < TOK; ++i) n[i] = 1.0f;
        if (!greedy) {
            if (vectors && v0 >= 0 && v0 + TOK <= V) {
#pragma unroll
                for (int h = 0; h < TOK; h += 4) {
                    const float4 w = *reinterpret_cast<const float4*>(q + v0 + h);
                    n[h] = w.x, n[h + 1] = w.y, n[h + 2] = w.z, n[h + 3] = w.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < TOK; ++i)
                    if (v0 + i >= 0 && v0 + i < V) n[i] = q[v0 + i];
            }
        }
#pragma unroll
        for (int h = 0; h < TOK; h += VEC) {
            float part[VEC];
            load_vector<T, VEC, RULES>(in, v0 + h, V, r, words + j + h, part);
#pragma unroll
            for (int i = 0; i < VEC; ++i) z[h + i] = part[i];
        }
        // over_temperature() with one branch a turn
        float a[TOK], most = -INFINITY;
        bool plain = true;
#pragma unroll
        for (int i = 0; i < TOK; ++i) a[i] = z[i] * inv, plain = plain && fabsf(a[i]) < 1e37f;
        if (plain) {
#pragma unroll
            for (int i = 0; i < TOK; ++i) z[i] = fmaf(fmaf(-a[i], t, z[i]), inv, a[i]);
        } else {
#pragma unroll 1
            for (int i = 0; i < TOK; ++i) {
                float y = 0.0f;
#pragma unroll
                for (int k = 0; k < TOK; ++k) y = k == i ? z[k] : y;  // (no indexed registers)
                y = over_temperature(y, t, inv);
#pragma unroll
                for (int k = 0; k < TOK; ++k) z[k] = k == i ? y : z[k];
            }
        }
#pragma unroll
        for (int i = 0; i < TOK; ++i) most = fmaxf(most, z[i]);
        if (most > x.max) {
            const float f = fast_exp(x.max - most);  // (0 the first time)
            x.score *= f, small = (small + (float)ones) * f, ones = 0;
            x.max = most;
#pragma unroll
            for (int i = TOK - 1; i >= 0; --i)
                if (z[i] == most) x.top = v0 + i;  // (the first of them)
        }
        if ((greedy && !sums) || x.max == -INFINITY) continue;
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const float e = fast_exp(z[i] - x.max);  // (0 of what is masked or not there)
            if (sums) {
                if (e == 1.0f) ++ones;
                else small += e;
            }
            const float score = race_score(e, n[i]);
            if (score > x.score) x.score = score, x.index = v0 + i, x.z = z[i];  // (tokens come in order)
        }
    }
    x.sum = (double)ones + (double)small;
    if (x.index == 0x7fffffff) x.score = -1.0f;
    // the CTA's, relative to its largest value
    float m = x.max;
    int top = x.top;
    block_max_index(m, top, s);
    const float f = x.max == -INFINITY ? 0.0f : expf(x.max - m);
    x.sum *= (double)f, x.max = m, x.top = top;
    if (x.index != 0x7fffffff) x.score *= f;
    x = block_part(x, s);
    cluster_wait();
    answer(x, greedy, s, cl, token + row, sums ? logprob + row : nullptr);
}

// Rows with filters.  The cuts are found by counts in 1024 bins of m - z (and by what the bins weigh, estimated), which single out a
// window of some hundred tokens; those alone are sorted, by the first CTA, with exact masses.  A row is in shared memory from the first pass
// on.  Some 20 steps that wait for one another (barriers of CTA and cluster, a sort) bound it, for many rows the same with two CTAs an SM.  Device us, 65536
// tokens fp16 with log-probability, one row / 64 / 256 rows: top-k 50 15.6 / 23.5 / 80, and with top-p the same; top-p 0.9 where 24 tokens are
// likely 16 / 24 / 83; top-p 0.9 of normal logits (2400 tokens kept) 21 / 34 / 124; min-p 8.7 / 15 / 54; a flat row, which no
// window holds, 47 / 94 / 350.
template <typename T, bool RULES>
__global__ void __launch_bounds__(lg::THREADS, 2) filter_kernel(const T* __restrict__ logits, int64_t ld, const rwkv7_logit_rules rules,
                                                                const rwkv7_draw_params draw, const float* __restrict__ noise, int64_t noise_ld,
                                                                long long* __restrict__ token, float* __restrict__ logprob, int V, int slice) {
    using namespace lg;
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    float* zs = reinterpret_cast<float*>(smem + FILTER_SHARED);
    cg::cluster_group cl = cg::this_cluster();
    constexpr int VEC = 16 / sizeof(T);
    const int C = cl.num_blocks(), rank = cl.block_rank();
    const int64_t row = blockIdx.x / C;
    const T* in = logits + row * ld;
    const int first = rank * slice - (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);
    if (threadIdx.x < 4) s.list_n[threadIdx.x] = 0;
    for (int b = threadIdx.x; b < BINS; b += THREADS) s.count[b] = 0, s.owned[b] = 0;
    cluster_arrive_relaxed();  // this CTA runs: the others may write into its shared memory
    grid_dependency_wait();
    grid_launch_dependents();
    const Draw d = row_draw(draw, noise != nullptr, row, V);
    const int k = d.k;
    const bool by_k = d.by_k, by_p = d.by_p;
    const float* q = noise + row * noise_ld;
    float m;
    int top;
    load_row<T, RULES>(in, first, V, slice, rules, row, d, zs, m, top);
    block_max_index(m, top, s);
    cluster_wait();
    row_max(m, top, s, cl);
    const float least = d.min_p > 0.0f ? d.min_p : 0.0f;
    Cut cut_k{0xffffffffu, 0x7fffffff, 0, false}, cut_p{0xffffffffu, 0x7fffffff, 0, false};
    if ((by_k || by_p) && m != -INFINITY) {
        // counts by distance from the largest value; every CTA sums up the bins it owns and reads the others' from their owners
        double sum = 0.0;
        int ones = 0;  // counted apart, as in finish()
        for (int j = threadIdx.x * VEC; j < slice; j += THREADS * VEC) {
#pragma unroll
            for (int h = 0; h < VEC; h += 4) {
                const float4 w = *reinterpret_cast<const float4*>(zs + j + h);
                const float z[4] = {w.x, w.y, w.z, w.w};
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (z[i] != -INFINITY) atomicAdd(&s.count[linear_bin(m, z[i])], 1u);
                    const float e = fast_exp(z[i] - m);
                    if (e == 1.0f) ++ones;
                    else part += e;
                }
                sum += (double)part;
            }
        }
        sum = block_add(sum + (double)ones, s.warp_sum);  // (its barriers also end the counting)
        const int per = BINS / C;
        for (int b = threadIdx.x; b < BINS; b += THREADS)
            if (s.count[b]) atomicAdd(&cl.map_shared_rank(&s, b / per)->owned[b], s.count[b]);
        if ((int)threadIdx.x < C) cl.map_shared_rank(&s, threadIdx.x)->sum_of[rank] = sum;
        cl.sync();
        double all = 0.0;
        for (int c = 0; c < C; ++c) all += s.sum_of[c];
        {
            const int b = 2 * threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            const uint2 n = *reinterpret_cast<const uint2*>(&cl.map_shared_rank(&s, b / per)->owned[b]);
            unsigned int c = n.x + n.y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned int t = __shfl_up_sync(0xffffffffu, c, o);
                if (lane >= o) c += t;
            }
            if (lane == 31) s.warp_count[warp] = c;
            if (threadIdx.x == 0) s.reach = BINS - 1;
            __syncthreads();
            for (int w = 0; w < warp; ++w) c += s.warp_count[w];
            s.upto[b] = c - n.y, s.upto[b + 1] = c;
            if (c - n.x - n.y <= FEW && c > FEW) s.reach = c - n.y > FEW ? b - 1 : b;
            __syncthreads();
        }
        const double share = d.p > 0.0f ? (double)d.p : 0.0;
        u64 target_p = share_of(share * MASS_UNIT, all);
#pragma unroll 1
        for (int stage = by_k && (unsigned int)k < s.upto[BINS - 1] ? 0 : 1; stage < (by_p ? 2 : 1); ++stage) {
            if (stage == 1 && cut_k.found) target_p = share_of(share, (double)cut_k.mass);
            // The last cut's list is short rather than whole: us of one row, top-k 500 / 900 with the whole list 20.2 / 23.4, around the cut 17.7 /
            // 18.0 (64 rows 33.8 / 37.0, 28.6 / 29.2), equal up to 128 tokens.  For top-k before top-p it is whole where that is possible, which
            // saves the second list: top-k 500 then top-p one row 20.2, two lists 26.7.
            const bool last = stage == 1 || !by_p;
            const unsigned int room = last ? 128 : LIST;
            choose_window(s, stage == 0 ? (unsigned int)k : 0u, (float)((double)target_p / MASS_UNIT), (float)all, room);
            // where the descent looks first if there is no list
            const int cut_bin = s.bin >> 2;
            int r0 = stage == 0 ? cut_bin : max(cut_bin - 2, 0), r1 = stage == 0 ? cut_bin : min(cut_bin + 2, BINS - 1);
            bool done = false;
#pragma unroll 1
            for (int turn = 2 * stage; turn < 2 * stage + 2 && !done; ++turn) {
                const int w0 = s.window_first, w1 = s.window_last;
                if (w0 > w1) break;
                // (on a list that holds all that top-k keeps the first CTA finds the masses itself)
                const bool masses = by_p && !(stage == 0 && w0 == 0);
                const unsigned int tokens = s.upto[w1] - (w0 ? s.upto[w0 - 1] : 0);
                // with the last cut in the window all above is kept, and what is kept of the list the first CTA finds: no other pass is needed
                const bool race = last && w0;
                if (race) race_above<VEC>(slice, first, m, least, q);
                gather<VEC>(zs, slice, first, m, s, cl, turn, cut_k.key, masses, tokens <= 128);
                u64 above = 0, listed = 0;
                for (int c = 0; masses && c < C; ++c) above += s.mass_of[turn][0][c], listed += s.mass_of[turn][1][c];
                // (by count the window is right; by mass the exact one has to agree, or everything is on the list)
                const bool right = stage == 0 || (above < target_p && above + listed >= target_p) || (w0 == 0 && w1 == BINS - 1);
                if (right && (w0 == 0 || last) && rank) return;
                if (right && rank == 0) {
                    const int n = (int)(s.upto[w1] - (w0 ? s.upto[w0 - 1] : 0));
                    sort_list(s.list, n);
                    const unsigned int above_count = w0 ? s.upto[w0 - 1] : 0;
                    const unsigned int key_k = stage == 0 ? (unsigned int)(s.list[k - (int)above_count - 1] >> 32) : cut_k.key;
                    const int kept = cut_k.found || stage == 0 ? places_upto(s.list, n, key_k) : n;
                    const Places o = weigh_list(s.list, kept, m, above, s);
                    if (w0 == 0 || last) {
                        const int i0 = threadIdx.x * 2;
                        const u64 target = !by_p ? ~0ull : stage == 0 ? share_of(share, (double)o.total) : target_p;
                        Part best{0.0, m, -1.0f, 0.0f, top, 0x7fffffff};
                        u64 before = o.before;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (i0 + i < kept && before < target && o.e[i] >= least) {
                                const int v = (int)(unsigned int)s.list[i0 + i];
                                const float score = race_score(o.e[i], q[v]);
                                if (better(score, v, best.score, best.index)) best.score = score, best.index = v, best.z = o.z[i];
                            }
                            before += o.w[i];
                        }
                        best = block_part(best, s);
                        if (threadIdx.x == 0) {
                            for (int c = 0; race && c < C; ++c) {
                                const Part& x = s.part[c];
                                if (better(x.score, x.index, best.score, best.index)) best.score = x.score, best.index = x.index, best.z = x.z;
                            }
                            const bool drawn = best.index != 0x7fffffff;  // (noise of NaN alone: the most likely token)
                            token[row] = drawn ? best.index : top;
                            if (logprob) logprob[row] = ((drawn ? best.z : m) - m) - log_sum(all);
                        }
                        return;
                    }
                    // top-k's cut to every CTA, for top-p
                    if ((int)threadIdx.x < C)
                        cl.map_shared_rank(&s, threadIdx.x)->cut = Cut{(unsigned int)(s.list[kept - 1] >> 32), 0x7fffffff, o.total, true};
                }
                if (right) {
                    cl.sync();
                    cut_k = s.cut;
                    done = true;
                } else {  // the cut lies in a bin before the window, or after it: the window beside it, once
                    const bool before = above >= target_p;
                    const int bin = before ? w0 - 1 : min(w1 + 1, BINS - 1);
                    r0 = before ? max(bin - 3, 0) : bin, r1 = before ? bin : min(bin + 3, BINS - 1);
                    __syncthreads();
                    place_window(s, bin, kAround, false, room);
                }
            }
            if (!done) {
                const Cut cut = descend(zs, slice, first, m, s, cl, stage == 1, stage == 0 ? (u64)k : target_p, r0, r1);
                (stage == 0 ? cut_k : cut_p) = cut;
            }
        }
    }
    const unsigned int key = cut_k.key < cut_p.key ? cut_k.key : cut_p.key;
    finish<VEC>(slice, first, m, top, d.greedy, q, token + row, logprob ? logprob + row : nullptr,
                [key, least, at_key = cut_p.key, from = cut_p.index](float z, int v, float e) {
                    const unsigned int kk = down_key(z);
                    return kk <= key && e >= least && !(kk == at_key && v >= from);
                });
}

}  // namespace rwkv7

using namespace rwkv7;

static int check_rules(const char* what, const rwkv7_logit_rules* r) {
    RWKV7_REQUIRE(r != nullptr, RWKV7_ERR_INVALID, "%s: null rules", what);
    RWKV7_REQUIRE(r->history >= 0, RWKV7_ERR_INVALID, "%s: negative history", what);
    RWKV7_REQUIRE(r->history <= (1 << 30), RWKV7_ERR_UNSUPPORTED, "%s: at most 2^30 tokens of history (got %d)", what, r->history);
    RWKV7_REQUIRE(r->tokens == nullptr || r->tokens_ld >= r->history, RWKV7_ERR_INVALID, "%s: the history's stride is shorter than a row", what);
    return RWKV7_OK;
}

extern "C" int rwkv7_process_logits(const void* logits, int64_t ld, const rwkv7_logit_rules* rules, void* out, int64_t out_ld, int B, int V,
                                    int dtype, void* stream) {
    RWKV7_REQUIRE(B > 0 && V > 0, RWKV7_ERR_INVALID, "process_logits: sizes must be positive");
    RWKV7_REQUIRE(B <= 65535, RWKV7_ERR_UNSUPPORTED, "process_logits: at most 65535 rows a call (got %d)", B);
    RWKV7_REQUIRE(logits && out, RWKV7_ERR_INVALID, "process_logits: null pointer");
    RWKV7_REQUIRE(ld >= V && out_ld >= V, RWKV7_ERR_INVALID, "process_logits: a row stride is shorter than a row");
    RWKV7_REQUIRE(V <= (1 << 30), RWKV7_ERR_UNSUPPORTED, "process_logits: at most 2^30 tokens (got %d)", V);
    if (int e = check_rules("process_logits", rules)) return e;
    // Tokens a CTA, a power of two made even over the row: few, so that a row or two spread over the GPU, more where the CTAs are
    // many all the same and every one of them reads its row's history.  us, 65536 tokens, 1024 / 2048 / 4096 / 8192 a CTA (of 512 threads the last): one
    // row, 300 of history 3.3 / 3.8 / 4.9 / 6.0; 16 rows, 1000 7.0 / 6.2 / 6.6 / 7.4; 64 rows, 512 16.9 / 13.1 / 12.2 / 12.4; 64
    // rows, 4096 33.7 / 22.6 / 18.2 / 15.2; 256 rows, 300 53 / 34 / 26.7 / 28.5.
    const int most = rules->tokens && rules->history > 1024 ? 8192 : 4096;
    int slice = 1024;
    while (slice < most && ((int64_t)V + slice - 1) / slice * B > 512) slice *= 2;
    const int threads = slice < 8192 ? 256 : 512, slices = (V + slice - 1) / slice, places = V + 16 / (int)dtype_size(dtype) - 1;
    slice = ((places + slices - 1) / slices + 7) / 8 * 8;
    const size_t smem = rules->tokens ? slice * 4 : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        e = launch_programmatic(process_logits_kernel<T>, dim3(slices, B), dim3(threads), smem, st, static_cast<const T*>(logits), ld, *rules,
                                static_cast<T*>(out), out_ld, V, slice);
    });
    RWKV7_REQUIRE(e == cudaSuccess, RWKV7_ERR_CUDA, "process_logits: %s", cudaGetErrorString(e));
    return check_launch("process_logits_kernel");
}

extern "C" int rwkv7_sample_tokens(const void* logits, int64_t ld, const rwkv7_logit_rules* rules, const rwkv7_draw_params* draw,
                                   const float* noise, int64_t noise_ld, long long* token, float* logprob, int B, int V, int dtype,
                                   void* stream) {
    using namespace lg;
    RWKV7_REQUIRE(B > 0 && V > 0, RWKV7_ERR_INVALID, "sample_tokens: sizes must be positive");
    RWKV7_REQUIRE(logits && draw && token, RWKV7_ERR_INVALID, "sample_tokens: null pointer");
    RWKV7_REQUIRE(ld >= V && (!noise || noise_ld >= V), RWKV7_ERR_INVALID, "sample_tokens: a row stride is shorter than a row");
    RWKV7_REQUIRE(dtype >= RWKV7_F16 && dtype <= RWKV7_F32, RWKV7_ERR_INVALID, "sample_tokens: unknown dtype %d", dtype);
    if (int e = check_rules("sample_tokens", rules)) return e;
    const int vec = 16 / (int)dtype_size(dtype);
    const bool filters = noise && (draw->top_k || (draw->top_k_value > 0 && draw->top_k_value < V) || draw->top_p || draw->top_p_value < 1.0f ||
                                   draw->min_p || draw->min_p_value > 0.0f);
    // CTAs a row: 4096 tokens each at least, eight for the shortest way.  Where the rows fill the GPU all the same, fewer and larger
    // slices cost less: a CTA's barriers and reductions are as long as its tokens.  us, 65536 tokens, 2 / 4 / 8 CTAs, top-p: one row 24 / 18.6 /
    // 15.3, 64 24.5 / 24.0 / 40.8, 256 95 / 84 / 128; without filters: one row 12.9 / 8.4 / 6.1, 16 13.4 / 8.7 / 7.3, 64 13.5 / 10.9 /
    // 14.4, 256 36.0 / 43.2 / 57.5.
    const int most = B <= 32 ? MAX_CLUSTER : filters || B <= 100 ? MAX_CLUSTER / 2 : MAX_CLUSTER / 4;
    const int64_t places = (int64_t)V + vec - 1, shared = filters ? FILTER_SHARED : PICK_SHARED;  // a row may begin up to vec - 1 places into its first vector
    const auto slice_of = [&](int c) { return ((places + c - 1) / c + 7) / 8 * 8; };
    const bool kept = filters || rules->tokens;  // whether a slice takes its place in shared memory
    const auto fits = [&](int c) { return shared + slice_of(c) * 4 <= 227 * 1024; };  // (one limit for every form of the call)
    int C = 1;
    while ((C < most && V > 4096 * C) || (C < MAX_CLUSTER && !fits(C))) C *= 2;
    const int64_t slice = slice_of(C), smem = shared + (kept ? slice * 4 : 0);
    const bool ruled = rules->tokens || rules->bias || rules->allowed;
    RWKV7_REQUIRE(fits(C), RWKV7_ERR_UNSUPPORTED, "sample_tokens: a vocabulary of %d tokens does not fit the shared memory of a cluster", V);
    RWKV7_REQUIRE((int64_t)B * C < (1ll << 31), RWKV7_ERR_UNSUPPORTED, "sample_tokens: too many rows (%d)", B);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        auto kernel = filters ? (ruled ? filter_kernel<T, true> : filter_kernel<T, false>) : ruled ? pick_kernel<T, true> : pick_kernel<T, false>;
        const cudaError_t a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        RWKV7_REQUIRE(a == cudaSuccess, RWKV7_ERR_CUDA, "sample_tokens: %s", cudaGetErrorString(a));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(B * C));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = (size_t)smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = C, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = programmatic_launch_ok(st) ? 2 : 1;
        cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), ld, *rules, *draw, noise, noise_ld, token, logprob, V, (int)slice);
    });
    return check_launch(filters ? "filter_kernel" : "pick_kernel");
}
