// What is done to a row of logits between the head and the next token.
//
// Rules (both kernels), in fp32, z the logit of token v, c how often v was generated, seen whether it occurs in the history at all:
//   seen: z > 0 ? z / repetition : z * repetition;  then  z - frequency * c - presence * (c > 0) + bias[v];  not allowed: -inf.
// Draw (sample_kernel), z / temperature, m the row's largest value, e = exp(z - m):
//   top-k  keeps z >= the k-th largest (ties stay);
//   top-p  keeps, in descending order (of equal values the lowest index first), every token with less than p of the mass of the
//          top-k survivors before it; the first always;
//   min-p  keeps e >= min_p;
//   token  = argmax of e / noise over what is kept (noise: independent Exp(1) variates, which makes it a draw from the
//            renormalised distribution); temperature <= 0: argmax of z.  The lowest index wins a tie.
// A NaN is never drawn, +inf counts as the largest finite number; a row without any token gives -1.
//
// A history is counted in shared memory, a word a token of the slice that a CTA holds (bit 31: in the prompt; below: times
// generated): integer atomics, so the order does not matter.  Every sum that is not of integers runs in a fixed order, and
// masses that are added by atomics are 64-bit fixed point (2^-40): results repeat bit for bit.
#include <cooperative_groups.h>

#include "umma.cuh"

namespace cg = cooperative_groups;

namespace rwkv7 {
namespace lg {
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 512;            // of a histogram
constexpr float BIN_SCALE = 16.0f;   // first histogram: m - z in steps of 1/16, the last bin takes the rest
constexpr float MASS_UNIT = 1099511627776.0f;  // 2^40

struct Exchange {
    double sum;
    float value, z;
    int index;
};
struct Shared {
    unsigned int count[BINS];          // this CTA's histogram
    unsigned long long mass[BINS];
    unsigned int all_count[2][BINS];   // the cluster's: [0] the first level, [1] the refinements
    unsigned long long all_mass[2][BINS];
    Exchange ex[3][MAX_CLUSTER];       // one for each use: nothing is written again while a CTA may still read it
    Exchange warp_ex[WARPS];
    unsigned int ties[MAX_CLUSTER];
    unsigned int warp_ties[WARPS];
    // crossing of a scan
    int bin;
    unsigned int above_count, bin_count;
    unsigned long long above_mass, bin_mass, target;
    int index_cut;
};
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
__device__ __forceinline__ float apply_rules(const Row& r, float z, unsigned int word, int v) {
    if (word) {
        z = z > 0.0f ? z / r.repetition : z * r.repetition;
        const unsigned int c = word & 0x7fffffffu;
        z = __fsub_rn(__fsub_rn(z, __fmul_rn(r.frequency, (float)c)), c ? r.presence : 0.0f);
    }
    if (r.bias) z = __fadd_rn(z, r.bias[v]);
    if (r.allowed && !((r.allowed[v >> 5] >> (v & 31)) & 1)) z = -INFINITY;
    return z;
}

// counts the history's tokens in [first, first + n) into words[0, n); ids outside the vocabulary fall outside every slice
__device__ __forceinline__ void count_history(const rwkv7_logit_rules& r, int64_t row, int first, int n, unsigned int* words) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) words[i] = 0;
    __syncthreads();
    int len = r.lengths ? r.lengths[row] : r.history;
    len = len < r.history ? len : r.history;
    const int prompt = r.prompt_lengths ? r.prompt_lengths[row] : 0;
    for (int i = threadIdx.x; i < len; i += blockDim.x) {
        const int64_t id = r.tokens_i64 ? static_cast<const int64_t*>(r.tokens)[row * r.tokens_ld + i]
                                        : (int64_t) static_cast<const int32_t*>(r.tokens)[row * r.tokens_ld + i];
        const int64_t at = id - first;
        if (id >= 0 && at >= 0 && at < n) {
            if (i >= prompt) atomicAdd(&words[at], 1u);
            else atomicOr(&words[at], 0x80000000u);
        }
    }
    __syncthreads();
}

// ---------------------------------------------------------------- rules alone
// grid (slices, rows); a row of any alignment is walked in 16-byte vectors that begin up to 16 bytes before it
template <typename T>
__global__ void __launch_bounds__(256) process_logits_kernel(const T* logits, int64_t ld, const rwkv7_logit_rules rules, T* out,
                                                             int64_t out_ld, int V, int slice) {
    extern __shared__ unsigned int words[];
    constexpr int VEC = 16 / sizeof(T);
    const int64_t row = blockIdx.y;
    const T* in = logits + row * ld;
    T* o = out + row * out_ld;
    const int mis = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);  // elements before the row in its first vector
    const bool vec_out = (reinterpret_cast<uintptr_t>(o) / sizeof(T)) % VEC == (uintptr_t)mis;
    const int first = blockIdx.x * slice - mis;  // token of the slice's first place (may lie before the row)
    const Row r = row_rules(rules, row);
    if (r.history) count_history(rules, row, first, slice, words);
    for (int j = threadIdx.x * VEC; j < slice; j += blockDim.x * VEC) {
        const int v0 = first + j;
        if (v0 >= V) break;
        if (v0 >= 0 && v0 + VEC <= V) {
            const uint4 raw = *reinterpret_cast<const uint4*>(in + v0);
            const T* e = reinterpret_cast<const T*>(&raw);
            alignas(16) T res[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) res[i] = from_f<T>(apply_rules(r, to_f<T>(e[i]), r.history ? words[j + i] : 0u, v0 + i));
            if (vec_out) {
                *reinterpret_cast<uint4*>(o + v0) = *reinterpret_cast<const uint4*>(res);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[v0 + i] = res[i];
            }
        } else {
            for (int i = 0; i < VEC; ++i)
                if (v0 + i >= 0 && v0 + i < V) o[v0 + i] = from_f<T>(apply_rules(r, to_f<T>(in[v0 + i]), r.history ? words[j + i] : 0u, v0 + i));
        }
    }
}

// ---------------------------------------------------------------- the draw
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// the block's best (value, lowest index first) with its z, and the block's sum in warp order; valid in every thread
__device__ __forceinline__ lg::Exchange block_best(lg::Exchange x, lg::Shared& s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, x.value, o), z = __shfl_xor_sync(0xffffffffu, x.z, o);
        const int i = __shfl_xor_sync(0xffffffffu, x.index, o);
        x.sum += __shfl_xor_sync(0xffffffffu, x.sum, o);
        if (better(v, i, x.value, x.index)) x.value = v, x.index = i, x.z = z;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_ex[threadIdx.x >> 5] = x;
    __syncthreads();
    x = s.warp_ex[0];
    for (int w = 1; w < lg::WARPS; ++w) {
        const lg::Exchange y = s.warp_ex[w];
        x.sum += y.sum;
        if (better(y.value, y.index, x.value, x.index)) x.value = y.value, x.index = y.index, x.z = y.z;
    }
    return x;
}

// the cluster's, in rank order; `slot` is used once a row
__device__ __forceinline__ lg::Exchange cluster_best(lg::Exchange x, lg::Shared& s, int slot, cg::cluster_group& cl) {
    x = block_best(x, s);
    const int C = cl.num_blocks(), rank = cl.block_rank();
    if ((int)threadIdx.x < C) cl.map_shared_rank(&s, threadIdx.x)->ex[slot][rank] = x;
    cl.sync();
    x = s.ex[slot][0];
    for (int c = 1; c < C; ++c) {
        const lg::Exchange y = s.ex[slot][c];
        x.sum += y.sum;
        if (better(y.value, y.index, x.value, x.index)) x.value = y.value, x.index = y.index, x.z = y.z;
    }
    return x;
}

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
// the last key of bins 0 .. bin: linear_bin rises with the key, so a bisection between keys on both sides of the edge (the
// bin's rounded edge is off by less than 2^-22 of the operands) finds it exactly
__device__ __forceinline__ unsigned int last_key(float m, int bin) {
    if (bin == lg::BINS - 1) return down_key(-3.402823466e38f);
    const float edge = m - (float)(bin + 1) / lg::BIN_SCALE, slack = (fabsf(m) + 64.0f) * 1e-6f;
    unsigned int lo = down_key(fminf(m, edge + slack)), hi = down_key(fmaxf(edge - slack, -3.402823466e38f));
    while (lo < hi) {
        const unsigned int mid = lo + (hi - lo + 1) / 2;
        if (linear_bin(m, key_value(mid)) <= bin) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ unsigned long long fixed_mass(float e) { return __float2ull_rn(e * lg::MASS_UNIT); }

// the cluster's histogram of `bin_of(z)` (negative: not counted) into all_count / all_mass[level] of every CTA
template <typename F>
__device__ __forceinline__ void histogram(const float* zs, int slice, float m, lg::Shared& s, int level, cg::cluster_group& cl, F bin_of) {
    for (int b = threadIdx.x; b < lg::BINS; b += lg::THREADS) s.count[b] = 0, s.mass[b] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < slice; j += lg::THREADS) {
        const float z = zs[j];
        if (z == -INFINITY) continue;
        const int b = bin_of(z);
        if (b >= 0) {
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], fixed_mass(expf(z - m)));
        }
    }
    cl.sync();
    const int C = cl.num_blocks(), rank = cl.block_rank(), per = lg::BINS / C;
    for (int b = rank * per + threadIdx.x; b < (rank + 1) * per; b += lg::THREADS) {
        unsigned int n = 0;
        unsigned long long q = 0;
        for (int c = 0; c < C; ++c) {
            lg::Shared* o = cl.map_shared_rank(&s, c);
            n += o->count[b], q += o->mass[b];
        }
        for (int c = 0; c < C; ++c) {
            lg::Shared* o = cl.map_shared_rank(&s, c);
            o->all_count[level][b] = n, o->all_mass[level][b] = q;
        }
    }
    cl.sync();
}

__device__ __forceinline__ unsigned long long share_of(double share, unsigned long long mass) {
    const double want = ceil(share * (double)mass);
    return want < 1.0 ? 1ull : (unsigned long long)want;
}

// first bin at which count (or mass) above the range plus that of bins 0 .. b reaches the target; results in s (bin = -1: none).
// share > 0: the target is that share of all the mass, rounded up.
__device__ __forceinline__ void find_crossing(lg::Shared& s, int level, bool by_mass, unsigned long long target, double share,
                                              unsigned int base_count, unsigned long long base_mass) {
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int PER = lg::BINS / 32;
        const int lane = threadIdx.x;
        unsigned int n = 0;
        unsigned long long q = 0;
        for (int i = 0; i < PER; ++i) n += s.all_count[level][lane * PER + i], q += s.all_mass[level][lane * PER + i];
        unsigned int cn = n;
        unsigned long long cq = q;
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned int tn = __shfl_up_sync(0xffffffffu, cn, o);
            const unsigned long long tq = __shfl_up_sync(0xffffffffu, cq, o);
            if (lane >= o) cn += tn, cq += tq;
        }
        if (share > 0.0) target = share_of(share, __shfl_sync(0xffffffffu, cq, 31));
        if (lane == 0) s.target = target;
        cn += base_count, cq += base_mass;
        const bool reached = (by_mass ? cq : (unsigned long long)cn) >= target;
        const unsigned int who = __ballot_sync(0xffffffffu, reached);
        if (who == 0) {
            if (lane == 0) s.bin = -1;
        } else if (lane == __ffs(who) - 1) {
            unsigned int an = cn - n;
            unsigned long long aq = cq - q;
            for (int i = 0; i < PER; ++i) {
                const int b = lane * PER + i;
                const unsigned int bn = s.all_count[level][b];
                const unsigned long long bq = s.all_mass[level][b];
                if ((by_mass ? aq + bq : (unsigned long long)(an + bn)) >= target) {
                    s.bin = b, s.bin_count = bn, s.bin_mass = bq, s.above_count = an, s.above_mass = aq;
                    break;
                }
                an += bn, aq += bq;
            }
        }
    }
    __syncthreads();
}

struct Cut {
    unsigned int key;            // values with down_key <= key are kept
    int index;                   // of values with exactly this key only tokens below this one
    unsigned long long mass;     // of what the key keeps
};

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
    if (lane == 31) s.warp_ties[warp] = upto;
    if (threadIdx.x == 0) s.index_cut = 0x7fffffff;
    __syncthreads();
    unsigned int total = 0, at = upto - mine;
    for (int w = 0; w < lg::WARPS; ++w) {
        if (w < warp) at += s.warp_ties[w];
        total += s.warp_ties[w];
    }
    const int C = cl.num_blocks(), rank = cl.block_rank();
    if ((int)threadIdx.x < C) cl.map_shared_rank(&s, threadIdx.x)->ties[rank] = total;
    cl.sync();
    unsigned int ahead = 0;
    for (int c = 0; c < rank; ++c) ahead += s.ties[c];
    if (ahead >= need) return 0;  // an earlier slice has them all
    at += ahead;
    for (int j = j0; j < j1; ++j)
        if (zs[j] != -INFINITY && down_key(zs[j]) == key && at++ == need) s.index_cut = first + j;
    __syncthreads();
    return s.index_cut;
}

// The key at which the descending order reaches `target` tokens (or mass, or a share of all of it), from the first level's
// histogram down.  A range of keys that is kept as a whole ends the search; its last key is the cut.
__device__ __forceinline__ Cut find_cut(const float* zs, int slice, int first, float m, lg::Shared& s, cg::cluster_group& cl, bool by_mass,
                                        unsigned long long target, double share) {
    find_crossing(s, 0, by_mass, target, share, 0, 0);
    if (s.bin < 0) return Cut{0xffffffffu, 0x7fffffff, 0};  // (only by count: fewer tokens than k)
    target = s.target;
    unsigned int lo = s.bin == 0 ? down_key(m) : last_key(m, s.bin - 1) + 1, hi = last_key(m, s.bin);
    for (int level = 0;; ++level) {  // (32 bits of key in steps of 9: four refinements at most)
        const unsigned int above_count = s.above_count, count = s.bin_count;
        const unsigned long long above_mass = s.above_mass, mass = s.bin_mass;
        // a single token, or (by count) all of them: the range is kept as a whole
        if (count == 1 || lo == hi || (!by_mass && above_count + count == target) || level == 4) {
            Cut cut{hi, 0x7fffffff, above_mass + mass};
            if (by_mass && count > 1) {
                const unsigned long long each = mass / count, need = (target - above_mass + each - 1) / each;
                if (need < count) cut.index = tie_cut(zs, slice, first, hi, (unsigned int)need, s, cl);
            }
            return cut;
        }
        const int bits = 32 - __clz(hi - lo), shift = bits > 9 ? bits - 9 : 0;
        histogram(zs, slice, m, s, 1, cl, [&](float z) {
            const unsigned int k = down_key(z);
            return k >= lo && k <= hi ? (int)((k - lo) >> shift) : -1;
        });
        find_crossing(s, 1, by_mass, target, 0.0, above_count, above_mass);
        if (s.bin < 0) return Cut{hi, 0x7fffffff, above_mass + mass};
        lo += (unsigned int)s.bin << shift;
        const unsigned int end = lo + ((1u << shift) - 1);
        hi = end < hi ? end : hi;
    }
}

template <typename T>
__global__ void __launch_bounds__(lg::THREADS, 1) sample_kernel(const T* __restrict__ logits, int64_t ld, const rwkv7_logit_rules rules,
                                                             const rwkv7_draw_params draw, const float* __restrict__ noise, int64_t noise_ld,
                                                             long long* __restrict__ token, float* __restrict__ logprob, int V, int slice) {
    using namespace lg;
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    float* zs = reinterpret_cast<float*>(smem + (sizeof(Shared) + 15) / 16 * 16);
    cg::cluster_group cl = cg::this_cluster();
    constexpr int VEC = 16 / sizeof(T);
    const int C = cl.num_blocks(), rank = cl.block_rank();
    const int64_t row = blockIdx.x / C;
    const T* in = logits + row * ld;
    const int mis = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);
    const int first = rank * slice - mis;
    const Row r = row_rules(rules, row);
    const float temperature = noise ? param(draw.temperature, draw.temperature_value, row) : 0.0f;
    const bool greedy = !(temperature > 0.0f);
    const float divisor = greedy ? 1.0f : temperature;

    cluster_arrive_relaxed();  // this CTA runs: the others may write into its shared memory
    if (r.history) count_history(rules, row, first, slice, reinterpret_cast<unsigned int*>(zs));
    Exchange x{0.0, -INFINITY, 0.0f, 0x7fffffff};
    for (int j = threadIdx.x * VEC; j < slice; j += THREADS * VEC) {
        const int v0 = first + j;
        const bool whole = v0 >= 0 && v0 + VEC <= V;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (whole) raw = *reinterpret_cast<const uint4*>(in + v0);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int v = v0 + i;
            float z = -INFINITY;
            if (v >= 0 && v < V) {
                z = apply_rules(r, to_f<T>(whole ? e[i] : in[v]), r.history ? __float_as_uint(zs[j + i]) : 0u, v) / divisor;
                z = z == z ? fminf(z, 3.402823466e38f) + 0.0f : -INFINITY;  // (-0 becomes 0)
            }
            zs[j + i] = z;
            if (better(z, v, x.value, x.index)) x.value = z, x.index = v;
        }
    }
    cluster_wait();
    x = cluster_best(x, s, 0, cl);
    const float m = x.value;
    const int top = x.index;
    if (m == -INFINITY) {  // no token at all
        if (rank == 0 && threadIdx.x == 0) {
            token[row] = -1;
            if (logprob) logprob[row] = -INFINITY;
        }
        return;
    }
    Cut cut_k{0xffffffffu, 0x7fffffff, 0}, cut_p{0xffffffffu, 0x7fffffff, 0};
    const float min_p = param(draw.min_p, draw.min_p_value, row);
    if (!greedy) {
        const int k = draw.top_k ? draw.top_k[row] : draw.top_k_value;
        const float p = param(draw.top_p, draw.top_p_value, row);
        const bool by_k = k > 0 && k < V, by_p = p < 1.0f;
        if (by_k || by_p) {
            histogram(zs, slice, m, s, 0, cl, [&](float z) { return linear_bin(m, z); });
            if (by_k) cut_k = find_cut(zs, slice, first, m, s, cl, false, (unsigned long long)k, 0.0);
            // of the mass that top-k keeps, or of all
            const double share = p > 0.0f ? (double)p : 1e-300;
            if (by_p) cut_p = find_cut(zs, slice, first, m, s, cl, true, share_of(share, cut_k.mass), cut_k.mass ? 0.0 : share);
        }
    }
    const unsigned int key = cut_k.key < cut_p.key ? cut_k.key : cut_p.key;
    Exchange best{0.0, -1.0f, 0.0f, 0x7fffffff};
    const float* q = noise + row * noise_ld;
    for (int j = threadIdx.x; j < slice; j += THREADS) {
        const float z = zs[j];
        if (z == -INFINITY) continue;
        const float e = expf(z - m);
        best.sum += (double)e;  // (a sure token's log-probability is all in the small terms)
        if (greedy) continue;
        const unsigned int k = down_key(z);
        const int v = first + j;
        if (k <= key && e >= min_p && !(k == cut_p.key && v >= cut_p.index)) {
            const float score = e / q[v];
            if (better(score, v, best.value, best.index)) best.value = score, best.index = v, best.z = z;
        }
    }
    best = cluster_best(best, s, 1, cl);
    if (rank == 0 && threadIdx.x == 0) {
        const bool drawn = !greedy && best.index != 0x7fffffff;  // (noise of NaN alone: the most likely token)
        token[row] = drawn ? best.index : top;
        if (logprob) logprob[row] = (float)((double)((drawn ? best.z : m) - m) - log(best.sum));
    }
}

}  // namespace rwkv7

using namespace rwkv7;

static int check_rules(const char* what, const rwkv7_logit_rules* r) {
    RWKV7_REQUIRE(r != nullptr, RWKV7_ERR_INVALID, "%s: null rules", what);
    RWKV7_REQUIRE(r->history >= 0, RWKV7_ERR_INVALID, "%s: negative history", what);
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
    const int slice = 8192;
    const size_t smem = rules->tokens ? slice * 4 : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        const int vec = 16 / sizeof(T);
        process_logits_kernel<T><<<dim3((V + vec - 1 + slice - 1) / slice, B), 256, smem, st>>>(static_cast<const T*>(logits), ld, *rules,
                                                                                                static_cast<T*>(out), out_ld, V, slice);
    });
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
    int C = 1;
    while (C < MAX_CLUSTER && V > 4096 * C) C *= 2;
    const int64_t places = (int64_t)V + vec - 1;  // a row may begin up to vec - 1 places into its first vector
    const int64_t slice = ((places + C - 1) / C + vec - 1) / vec * vec;
    const int64_t smem = (sizeof(Shared) + 15) / 16 * 16 + slice * 4;
    RWKV7_REQUIRE(smem <= 227 * 1024, RWKV7_ERR_UNSUPPORTED, "sample_tokens: a vocabulary of %d tokens does not fit the shared memory of a cluster", V);
    RWKV7_REQUIRE((int64_t)B * C < (1ll << 31), RWKV7_ERR_UNSUPPORTED, "sample_tokens: too many rows (%d)", B);
    RWKV7_DISPATCH_DTYPE(dtype, T, {
        auto kernel = sample_kernel<T>;
        const cudaError_t a = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        RWKV7_REQUIRE(a == cudaSuccess, RWKV7_ERR_CUDA, "sample_tokens: %s", cudaGetErrorString(a));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(B * C));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = (size_t)smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = C, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), ld, *rules, *draw, noise, noise_ld, token, logprob, V, (int)slice);
    });
    return check_launch("sample_kernel");
}
