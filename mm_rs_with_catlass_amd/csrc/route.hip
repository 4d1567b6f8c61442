// The router: which experts a token goes to, with what shares, the shares' gradient, and the rows' order by expert.
//
//   score p_e = softmax(l)_e or s(l_e); the `top` largest of p_e + b_e, in the topGroups groups whose best one or two sum to most; share = scale p_c (/ sum of the chosen p).
//
// A token's experts lie on 16 or 64 lanes, a group of them on a power of two of those, up to 32 a lane: four tokens a wave where 16 lanes hold them (16384 tokens
// of 256 experts, biased, 12 us; twice that with a wave for each token).  An expert's rank is one 64-bit number, its key: a double whose last ten bits are the expert's index, counted so that of equal scores
// the lower index is the larger key.  Maxima of doubles, as fast here as those of floats, then order scores and ties alike, and nothing has to be carried along with a
// score.  Where the order is that of the logits (no bias, no sums of scores) a key holds all of a logit's bits; else it is the score in 64 bits, whose first 42 bits count: which of
// two experts is ahead is a matter of more bits than fp32 has, as one of a prompt's 10^5 choices is decided by less than 2^-24 now and then.
// Every lane sorts its keys once (odd-even merge sort: Batcher, AFIPS 1968); then the largest of the lanes' first keys is taken `top` times.
//
// Bound by its 64-bit instructions where there are many tokens: us a call, three or more sets of logits in turn: 16384 of 256 experts in groups, biased, 12 (1200 instructions a wave, 74 % of the time; the logits alone
// would take 3.5), by the logits alone 8, and 50 us with the library's exponential and division, a load for each bias and the compiler's way of moving up a sorted list; 32 tokens of 64 experts 3.0 us on the GPU.  512
// experts, top 10: 19 us, in groups and biased 27.
#include <hip/hip_runtime.h>

#include <utility>

#include "layer_args.h"
#include "rows_device.h"

namespace catcoc {

namespace {

constexpr double kMostKey = 0x1p1000;     // infinity and NaN count as this,
constexpr double kNone = -0x1p1000;       // and what is not to be had as this, or less by its index
constexpr uint32_t kIndexBits = 1023;

// An exchange between lanes of a row of 16.
template <int CTRL>
__device__ __forceinline__ float lane_turn(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}

template <int CTRL>
__device__ __forceinline__ double lane_turn(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

template <typename F, int... I>
__device__ __forceinline__ void turns(F f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, 0x121 + I>{}), ...);   // row_ror:1 to 15
}

// f with each of the 15 turns of a row of 16 lanes.
template <typename F>
__device__ __forceinline__ void each_other_lane(F f)
{
    turns(f, std::make_integer_sequence<int, 15>{});
}

// f over the values of LANES lanes, in all of them, in an order that is always the same.
template <int LANES, typename T, typename F>
__device__ __forceinline__ T over_lanes(T v, F f)
{
    v = f(v, lane_turn<0x128>(v));   // row_ror:8, 4, 2, 1
    v = f(v, lane_turn<0x124>(v));
    v = f(v, lane_turn<0x122>(v));
    v = f(v, lane_turn<0x121>(v));
    if constexpr (LANES == 64) {
        v = f(v, __shfl_xor(v, 16));
        v = f(v, __shfl_xor(v, 32));
    }
    return v;
}

template <int LANES, typename T>
__device__ __forceinline__ T lanes_max(T v)
{
    return over_lanes<LANES>(v, [](T a, T b) { return __builtin_elementwise_max(a, b); });
}

template <int LANES, typename T>
__device__ __forceinline__ T lanes_sum(T v)
{
    return over_lanes<LANES>(v, [](T a, T b) { return a + b; });
}

// (A NaN is no operand of a minimum: what is left is the other one.)
__device__ __forceinline__ double with_index(double k, uint32_t index)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, __builtin_elementwise_max(__builtin_elementwise_min(k, kMostKey), kNone));
    const uint32_t hi = (uint32_t)(b >> 32), counted = ~(index ^ (uint32_t)((int32_t)hi >> 31));   // down from 1023, below zero up from 0
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | (((uint32_t)b & ~kIndexBits) | (counted & kIndexBits)));
}

__device__ __forceinline__ double without_index(double k) { return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, k) & ~(uint64_t)kIndexBits); }

__device__ __forceinline__ uint32_t index_of(double k)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, k);
    return ((uint32_t)b ^ ~(uint32_t)((int32_t)(b >> 32) >> 31)) & kIndexBits;
}

__device__ __forceinline__ void in_order(double &a, double &b)
{
    const double hi = __builtin_elementwise_max(a, b), lo = __builtin_elementwise_min(a, b);
    a = hi;
    b = lo;
}

// Largest first.
template <int V>
__device__ __forceinline__ void sort_keys(double (&k)[V])
{
#pragma unroll
    for (int p = 1; p < V; p <<= 1)
#pragma unroll
        for (int q = p; q > 0; q >>= 1)
#pragma unroll
            for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) in_order(k[i + j], k[i + j + q]);
}

__device__ __forceinline__ float widen1(uint32_t h, uint32_t type)
{
    return type == DT_BF16 ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (unsigned short)h);
}

__device__ __forceinline__ float logit_at(const void *x, size_t at, uint32_t type)
{
    return type == 0 ? ((const float *)x)[at] : widen1(((const unsigned short *)x)[at], type);
}

// Value i of a lane that is `part` of a group's lanes is the group's expert place_in_group(): consecutive lanes hold consecutive pieces of P.  Pieces of four, with which a
// wave's accesses lie beside each other, where there is little but them (gradients of 16384 tokens of 256 experts 10 us, a third more with a lane's values in one piece), one
// piece where there are few registers left (the choice of the same a quarter more with pieces of four).
template <int P>
__device__ __forceinline__ uint32_t place_in_group(uint32_t part, uint32_t lanes, int i)
{
    return ((uint32_t)(i / P) * lanes + part) * P + (uint32_t)(i % P);
}

// A lane's logits of a group of `size` that begins at `at`, -inf for those there are not.
template <int P, int V>
__device__ __forceinline__ void load_logits(const void *x, size_t at, uint32_t part, uint32_t lanes, uint32_t size, uint32_t type, float (&v)[V])
{
#pragma unroll
    for (int c = 0; c < V / P; ++c) {
        const uint32_t o = place_in_group<P>(part, lanes, c * P);
        if (type == 0) {
            const float *p = (const float *)x + at + o;
            if (o + P <= size) __builtin_memcpy(&v[c * P], p, P * 4);
            else {
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)P; ++i) v[c * P + i] = o + i < size ? p[i] : -__builtin_huge_valf();
            }
        } else {
            const unsigned short *p = (const unsigned short *)x + at + o;
            unsigned short h[P];
            if (o + P <= size) __builtin_memcpy(h, p, P * 2);
            else {
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)P; ++i) h[i] = o + i < size ? p[i] : 0;
            }
#pragma unroll
            for (uint32_t i = 0; i < (uint32_t)P; ++i) v[c * P + i] = o + i < size ? widen1(h[i], type) : -__builtin_huge_valf();
        }
    }
}

// e^x to 2^-44.4 of it, |x| <= 700 (2^-45.3 to 100: the one constant for ln 2 is off by 2^-54 of it, n times over): 2^n e^r with |r| <= ln 2 / 2 and e^r as the polynomial
// that meets it at ten Chebyshev nodes (2^-45.6).  Beside 1.5 2^52 a number is
// a whole one, n the last bits of the sum.
__device__ __forceinline__ double exp64(double x)
{
    const double t = __builtin_fma(x, 0x1.71547652b82fep+0, 0x1.8p52), n = t - 0x1.8p52, r = __builtin_fma(n, -0x1.62e42fefa39efp-1, x);
    double p = 0x1.72e107c874de9p-19;
    p = __builtin_fma(p, r, 0x1.a17df0d914d6cp-16);
    p = __builtin_fma(p, r, 0x1.a01994c849582p-13);
    p = __builtin_fma(p, r, 0x1.6c162bb7d965cp-10);
    p = __builtin_fma(p, r, 0x1.11111123bf154p-7);
    p = __builtin_fma(p, r, 0x1.55555588b8403p-5);
    p = __builtin_fma(p, r, 0x1.5555555550d88p-3);
    p = __builtin_fma(p, r, 0x1.ffffffffe74f1p-2);
    p = __builtin_fma(p, r, 0x1.0000000000006p+0);
    p = __builtin_fma(p, r, 0x1.000000000003dp+0);
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, t) << 52));
}

// The sigmoid to 2^-44 of it; logits further than 700 from zero count as that.  A reciprocal is the instruction's, 2^-24 off, and a step of Newton's.
__device__ __forceinline__ double sigmoid64(float x)
{
    const double d = 1.0 + exp64(-(double)__builtin_amdgcn_fmed3f(x, -700.f, 700.f)), r = __builtin_amdgcn_rcp(d);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// What an expert's share is made of, from its logit: of the softmax e^(l - most), of the sigmoid s(l), where it is only to be compared with that of the largest logit,
// `most`, and that is not positive, e^(l - most) / (1 + e^l) in its place: s(l) itself could be 0 for all of them.
__device__ __forceinline__ float weight_of(float l, float most, bool sigmoid, bool compared)
{
    if (!sigmoid) return expf(l - most);
    return compared && most <= 0.f ? expf(l - most) / (1.f + expf(l)) : 1.f / (1.f + expf(-l));
}

}  // namespace

template <int LANES, int V>
__global__ void __launch_bounds__(256, LANES == 16 ? 4 : V <= 16 ? 3 : 2) route_kernel(const RouteArgs args)
{
    const uint32_t lane = threadIdx.x & 63u, l = lane % LANES;
    const uint64_t at = ((uint64_t)workgroup() * 4u + (threadIdx.x >> 6)) * (64 / LANES) + lane / LANES;
    if (at - lane / LANES >= args.tokens) return;   // (a wave without tokens)
    const size_t token = at < args.tokens ? at : args.tokens - 1u;   // (the last one once more, for nothing)
    const uint32_t each = args.experts / args.groups, slot = l / args.groupLanes, part = l % args.groupLanes;
    const uint32_t size = slot < args.groups ? each : 0u, first = size ? slot * each : 0u;   // the group's
    float v[V];
    load_logits<V, V>(args.logits, token * args.experts + first, part, args.groupLanes, size, args.type, v);

    float most = 0.f;
    if (!args.sigmoid) {
        most = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) most = __builtin_elementwise_max(most, v[i]);
        most = lanes_max<LANES>(most);
    }
    double k[V];
    float total = 0.f;   // of the softmax
    if (args.bias != nullptr || args.groupTop == 2) {
        bool odd = false;   // NaN, infinite, or not to be had
#pragma unroll
        for (int i = 0; i < V; ++i) odd |= !(__builtin_fabsf(v[i]) < __builtin_huge_valf());
        double r = 1.0;
        if (args.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) k[i] = sigmoid64(v[i]);
        } else {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                k[i] = exp64(__builtin_elementwise_max((double)v[i] - (double)most, -700.0));
                sum += k[i];
            }
            bool spoilt = !(most < __builtin_huge_valf());
            if (__any(odd)) {
#pragma unroll
                for (int i = 0; i < V; ++i) spoilt |= v[i] != v[i];
            }
            sum = lanes_sum<LANES>(spoilt ? (double)__builtin_nanf("") : sum);   // (of values not all of which are numbers: no score)
            total = (float)sum;
            r = 1.0 / sum;
        }
        float b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = 0.f;
        if (args.bias != nullptr) load_logits<V, V>(args.bias, first, part, args.groupLanes, size, 0, b);
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = __builtin_fma(k[i], r, (double)b[i]);
        if (__any(odd)) {
#pragma unroll
            for (int i = 0; i < V; ++i) k[i] = b[i] == -__builtin_huge_valf() ? kNone : v[i] > -__builtin_huge_valf() ? k[i] : (double)v[i];   // (a bias masks a score that is NaN)
        }
    } else {
        if (!args.sigmoid && !args.renormalize) {
#pragma unroll
            for (int i = 0; i < V; ++i) total += v[i] == -__builtin_huge_valf() ? 0.f : expf(v[i] - most);
            total = lanes_sum<LANES>(total);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = v[i] + 0.f;   // (-0 is 0)
    }
#pragma unroll
    for (int i = 0; i < V; ++i) k[i] = with_index(k[i], first + part * V + i);
    sort_keys<V>(k);

    bool out = false;   // of the groups that are chosen from
    if (args.topGroups < args.groups) {
        double a = k[0], b = V > 1 ? k[V > 1 ? 1 : 0] : kNone;   // the group's best two
        for (uint32_t by = 1; by < args.groupLanes; by <<= 1) {
            const double c = __shfl_xor(a, (int)by), d = __shfl_xor(b, (int)by);
            b = __builtin_elementwise_max(__builtin_elementwise_min(a, c), __builtin_elementwise_max(b, d));
            a = __builtin_elementwise_max(a, c);
        }
        double best = without_index(a);
        if (args.groupTop == 2 && b > kNone) best += without_index(b);   // (a group with one expert left goes by that one, as a group of one does)
        best = with_index(best, slot);
        uint32_t ahead = 0;   // how many groups are
        if constexpr (LANES == 16) {
            each_other_lane([&](auto turn) { ahead += lane_turn<decltype(turn)::value>(best) > best ? 1u : 0u; });   // (a group counts once for each of its lanes)
            out = ahead >= args.topGroups * args.groupLanes;
        } else {
            for (uint32_t g = 0; g < args.groups; ++g) ahead += __shfl(best, (int)(g * args.groupLanes), LANES) > best ? 1u : 0u;
            out = ahead >= args.topGroups;
        }
    }

    double mine = kNone;   // lane j: the j-th choice
    if constexpr (V <= 4) {
        if (out) {
#pragma unroll
            for (int i = 0; i < V; ++i) k[i] = kNone;
        }
        for (uint32_t j = 0; j < args.top; ++j) {
            const double next = lanes_max<LANES>(k[0]);
            if (l == j) mine = next;
            if (k[0] == next) {   // (a branch: as selects, the compiler makes an index of them and looks for it among all keys)
#pragma unroll
                for (int i = 0; i + 1 < V; ++i) k[i] = k[i + 1];
                k[V - 1] = kNone;
            }
        }
    } else {
        // A lane's first two keys are in registers, the others wait in LDS: moving 15 of them up in registers at each turn took a third of the kernel's instructions.
        __shared__ double keys[V + 1][256];
#pragma unroll
        for (int i = 2; i < V; ++i)
            if ((uint32_t)i <= args.top) keys[i][threadIdx.x] = k[i];
        keys[V][threadIdx.x] = kNone;
        double first_key = out ? kNone : k[0], second = out ? kNone : k[1];
        uint32_t at_key = out ? (uint32_t)V : 2u;   // the one behind the second
        for (uint32_t j = 0; j < args.top; ++j) {
            const double next = lanes_max<LANES>(first_key);
            if (l == j) mine = next;
            const bool taken = first_key == next;
            const double third = keys[at_key][threadIdx.x];
            first_key = taken ? second : first_key;
            second = taken ? third : second;
            at_key = umin(at_key + (taken ? 1u : 0u), (uint32_t)V);
        }
    }
    const bool on = mine > kNone;
    const uint32_t expert = on ? index_of(mine) : 0u;
    const float logit = on ? logit_at(args.logits, token * args.experts + expert, args.type) : -__builtin_huge_valf();
    if (args.renormalize) most = lanes_max<LANES>(logit);
    float share = on ? weight_of(logit, most, args.sigmoid, args.renormalize) : 0.f;
    if (args.renormalize) total = total == total ? lanes_sum<LANES>(share) : total;   // (a softmax with a NaN or an infinity in it has no other scores either)
    if (args.renormalize || !args.sigmoid) share /= total;
    if (l >= args.top || at >= args.tokens) return;
    args.choice[token * args.top + l] = on ? (int32_t)expert : -1;
    args.share[token * args.top + l] = on ? share * args.scale : 0.f;
}

// Between a wave's writes to LDS and its reads of other lanes' (LDS keeps a wave's accesses in order, the compiler knows of one lane's only).
__device__ __forceinline__ void wave_turn() { asm volatile("" ::: "memory"); }

// With w the shares without scale: dl_c = scale w_c (1 - s(l_c) where sigmoid) (g_c - sum of w g where they are shares of a sum); the softmax of all experts: dl_e = scale p_e (g_e - sum of p g).
template <int LANES, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs args)
{
    constexpr int P = V < 4 ? V : 4;
    const uint32_t lane = threadIdx.x & 63u, l = lane % LANES;
    const uint64_t at = ((uint64_t)workgroup() * 4u + (threadIdx.x >> 6)) * (64 / LANES) + lane / LANES;
    if (at - lane / LANES >= args.tokens) return;
    const size_t token = at < args.tokens ? at : args.tokens - 1u;
    const bool all = !args.sigmoid && !args.renormalize;   // every expert's logit moves the shares
    float v[V], most = 0.f, total = 1.f;
    if (all) {
        load_logits<P, V>(args.logits, token * args.experts, l, LANES, args.experts, args.type, v);
        most = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) most = __builtin_elementwise_max(most, v[i]);
        most = lanes_max<LANES>(most);
        total = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = v[i] == -__builtin_huge_valf() ? 0.f : expf(v[i] - most);
            total += v[i];
        }
        total = lanes_sum<LANES>(total);
    }
    const int32_t chosen = l < args.top ? args.chosen[token * args.top + l] : -1;
    const bool on = (uint32_t)chosen < args.experts;
    const float g = on ? args.dshare[token * args.top + l] * args.scale : 0.f;
    const float logit = on ? logit_at(args.logits, token * args.experts + (uint32_t)chosen, args.type) : -__builtin_huge_valf();
    if (args.renormalize) most = lanes_max<LANES>(logit);
    float w = on && logit != -__builtin_huge_valf() ? weight_of(logit, most, args.sigmoid, args.renormalize) : 0.f;
    if (args.renormalize) total = lanes_sum<LANES>(w);
    if ((args.renormalize || !args.sigmoid) && total > 0.f) w /= total;   // (no sum: no expert)
    const float sum = args.renormalize || all ? lanes_sum<LANES>(w * g) : 0.f;
    float d = w * (g - (all ? 0.f : sum));
    if (args.sigmoid) d *= 1.f / (1.f + expf(logit));
    if (all) {
        const float r = total > 0.f ? -sum / total : 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= r;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
    }
    if constexpr (V <= 4) {
        for (uint32_t j = 0; j < args.top; ++j) {   // (an expert that is chosen twice gets both)
            const uint32_t to = (uint32_t)__shfl(chosen, (int)j, LANES) - l * V;
            const float more = __shfl(d, (int)j, LANES);
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) v[i] += to == i ? more : 0.f;
        }
    } else {
        // Through LDS, where a choice finds its expert's place; an expert that is chosen twice gets both from each of its choices.
        __shared__ float rows[256 * V];
        float *const row = rows + (threadIdx.x - l) * V;
        float more = 0.f;
        for (uint32_t j = 0; j < args.top; ++j) {
            const int32_t other = __shfl(chosen, (int)j, LANES);
            const float part = __shfl(d, (int)j, LANES);
            more += other == chosen ? part : 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) row[place_in_group<P>(l, LANES, i)] = v[i];
        wave_turn();
        const uint32_t place = on ? (uint32_t)chosen : 0u;
        const float there = row[place] + more;
        wave_turn();
        if (on) row[place] = there;
        wave_turn();
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = row[place_in_group<P>(l, LANES, i)];
    }
    if (at >= args.tokens) return;
#pragma unroll
    for (int c = 0; c < V / P; ++c) {
        const uint32_t o = place_in_group<P>(l, LANES, c * P);
        if (o >= args.experts) continue;
        const size_t to = token * args.experts + o;
        if (args.type == 0) {
            float *p = (float *)args.dlogits + to;
            if (o + P <= args.experts) __builtin_memcpy(p, &v[c * P], P * 4);
            else {
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)P; ++i)
                    if (o + i < args.experts) p[i] = v[c * P + i];
            }
        } else {
            unsigned short h[P], *p = (unsigned short *)args.dlogits + to;
#pragma unroll
            for (int i = 0; i < P; ++i)
                h[i] = args.type == DT_BF16 ? __builtin_bit_cast(unsigned short, (__bf16)v[c * P + i]) : __builtin_bit_cast(unsigned short, (_Float16)v[c * P + i]);
            if (o + P <= args.experts) __builtin_memcpy(p, h, P * 2);
            else {
#pragma unroll
                for (uint32_t i = 0; i < (uint32_t)P; ++i)
                    if (o + i < args.experts) p[i] = h[i];
            }
        }
    }
}

template <int LANES, int V, bool BACKWARD>
static int launch_route_kernel(const RouteArgs &a, hipStream_t stream)
{
    const uint64_t waves = (a.tokens + (uint64_t)(64 / LANES) - 1u) / (64 / LANES);
    const dim3 grid = grid_of((waves + 3) / 4, 256);
    if constexpr (BACKWARD) hipLaunchKernelGGL((route_backward_kernel<LANES, V>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((route_kernel<LANES, V>), grid, dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

// Lanes of a token, of a group in it, and values a lane, for `groups` groups of experts: 16 lanes where they hold it in 16 values each, else 64.  0 lanes: not on these.
struct RouteShape {
    uint32_t lanes, groupLanes, perLane;
};
static RouteShape route_shape(uint32_t experts, uint32_t top, uint32_t groups)
{
    uint32_t slots = 1;
    while (slots < groups) slots *= 2;
    const uint32_t size = experts / groups;
    for (uint32_t lanes = 16; lanes <= 64; lanes *= 4) {
        if (slots > lanes || top > lanes) continue;
        const uint32_t of = lanes / slots, n = (size + of - 1) / of;
        if (n <= (lanes == 16 ? 16u : 32u)) return {lanes, of, n};
    }
    return {0, 0, 0};
}

template <bool BACKWARD>
static int launch_route_shape(RouteArgs a, hipStream_t stream)
{
    const RouteShape s = route_shape(a.experts, a.top, BACKWARD ? 1u : a.groups);
    const uint32_t n = s.perLane;
    a.groupLanes = s.groupLanes;
    if (s.lanes == 16) {
        if (n <= 1) return launch_route_kernel<16, 1, BACKWARD>(a, stream);
        if (n <= 2) return launch_route_kernel<16, 2, BACKWARD>(a, stream);
        if (n <= 4) return launch_route_kernel<16, 4, BACKWARD>(a, stream);
        if (n <= 8) return launch_route_kernel<16, 8, BACKWARD>(a, stream);
        return launch_route_kernel<16, 16, BACKWARD>(a, stream);
    }
    if (n <= 2) return launch_route_kernel<64, 2, BACKWARD>(a, stream);
    if (n <= 8) return launch_route_kernel<64, 8, BACKWARD>(a, stream);
    if (n <= 16) return launch_route_kernel<64, 16, BACKWARD>(a, stream);
    if constexpr (!BACKWARD) return launch_route_kernel<64, 32, false>(a, stream);   // (groups in a number that is no power of two)
    return -1;
}

// Groups that the kernel can lay out: at most 64 of them.
bool can_route(uint32_t experts, uint32_t top, uint32_t groups)
{
    return route_shape(experts, top, groups).lanes != 0;
}

int launch_route(const RouteArgs &a, void *stream) { return launch_route_shape<false>(a, (hipStream_t)stream); }
int launch_route_backward(const RouteArgs &a, void *stream) { return launch_route_shape<true>(a, (hipStream_t)stream); }

// ---- rows by expert -----------------------------------------------------------------------------------------------------------------------
// A counting sort, stable: a wave counts how many of its consecutive rows go to each expert, the counts' sums over waves, blocks and experts are where its first
// row of each goes, and the rows follow in 64s, a row's place among them by how many lanes before it have the same expert.  Latencies bound it: 256 rows 3.2 us, 8192 to 128
// experts 5.4, 131072 9.2 (two launches of 2.9 and 6.5; the bytes would take 0.3).

namespace {

constexpr uint32_t kSortWaves = 16, kSortThreads = 64 * kSortWaves;

constexpr uint32_t kSortTurns = 4;   // times 64 rows that a wave asks for together
constexpr uint32_t kNoRow = 0xffffffffu;

// The experts of a wave's rows [first, first + 256) that are before `end`.
template <typename I>
__device__ __forceinline__ void load_experts(const SortArgs &args, uint32_t first, uint32_t end, uint32_t (&expert)[kSortTurns])
{
    I c[kSortTurns];
    const uint32_t at = first + (threadIdx.x & 63u);   // (below 2^31 + 2^8)
#pragma unroll
    for (uint32_t i = 0; i < kSortTurns; ++i) c[i] = ((const I *)args.choice)[umin(at + 64u * i, end - 1u)];
#pragma unroll
    for (uint32_t i = 0; i < kSortTurns; ++i) expert[i] = at + 64u * i >= end ? kNoRow : c[i] >= 0 && c[i] < (I)args.experts ? (uint32_t)c[i] : args.experts;
}

// How many of each wave's rows go to each expert.  `expert`: of its first 256 rows on the way in, of its last ones on the way out.
template <typename I, uint32_t MOST>
__device__ __forceinline__ void count_rows(const SortArgs &args, uint32_t (&count)[kSortWaves][MOST + 1], uint32_t begin, uint32_t end, uint32_t (&expert)[kSortTurns])
{
    for (uint32_t i = threadIdx.x; i < kSortWaves * (MOST + 1u); i += kSortThreads) (&count[0][0])[i] = 0;
    __syncthreads();
    uint32_t *const mine = count[threadIdx.x >> 6];
    for (uint32_t first = begin; first < end; first += 64u * kSortTurns) {
        if (first != begin) load_experts<I>(args, first, end, expert);
#pragma unroll
        for (uint32_t i = 0; i < kSortTurns; ++i)
            if (expert[i] != kNoRow) atomicAdd(&mine[expert[i]], 1u);
    }
    __syncthreads();
}

// How many of the rows [begin, end) go to each expert, added to `hist`.
template <typename I>
__device__ __forceinline__ void count_others(const SortArgs &args, uint32_t *hist, uint32_t begin, uint32_t end)
{
#pragma unroll 4
    for (uint32_t first = begin + (threadIdx.x >> 6) * 64u * kSortTurns; first < end; first += kSortThreads * kSortTurns) {
        uint32_t expert[kSortTurns];
        load_experts<I>(args, first, end, expert);
#pragma unroll
        for (uint32_t i = 0; i < kSortTurns; ++i)
            if (expert[i] < args.experts) atomicAdd(&hist[expert[i]], 1u);
    }
}

__device__ __forceinline__ void wave_rows(const SortArgs &args, uint32_t &begin, uint32_t &end)
{
    const uint32_t each = args.perBlock / kSortWaves;
    const uint64_t from = (uint64_t)blockIdx.x * args.perBlock + (threadIdx.x >> 6) * each;
    begin = (uint32_t)(from < args.rows ? from : args.rows);
    end = (uint32_t)(from + each < args.rows ? from + each : args.rows);
}

}  // namespace

template <typename I, uint32_t MOST>
__global__ void __launch_bounds__(kSortThreads) count_by_expert_kernel(const SortArgs args)
{
    __shared__ uint32_t count[kSortWaves][MOST + 1];
    uint32_t begin, end, expert[kSortTurns];
    wave_rows(args, begin, end);
    if (begin < end) load_experts<I>(args, begin, end, expert);
    count_rows<I, MOST>(args, count, begin, end, expert);
    if (threadIdx.x < args.experts) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) n += count[w][threadIdx.x];
        args.part[(size_t)blockIdx.x * args.experts + threadIdx.x] = n;
    }
}

template <typename I, uint32_t MOST>
__global__ void __launch_bounds__(kSortThreads) sort_by_expert_kernel(const SortArgs args)
{
    __shared__ uint32_t count[kSortWaves][MOST + 1];
    __shared__ uint32_t totals[kSortThreads], before[kSortThreads], sums[2][kSortWaves];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    uint32_t begin, end, n = 0, those = 0, expert[kSortTurns];
    wave_rows(args, begin, end);
    if (begin < end) load_experts<I>(args, begin, end, expert);
    // ---- thread e: rows of expert e, of all blocks (n) and of those before this one; the blocks' counts are read by as many threads an expert as there are
    const uint32_t wide = args.experts <= 64u ? 6u : 32u - (uint32_t)__builtin_clz(args.experts - 1u);
    if (args.part != nullptr) {
        const uint32_t e = threadIdx.x & ((1u << wide) - 1u);
        uint32_t all = 0, some = 0;
        if (e < args.experts) {
#pragma unroll 16
            for (uint32_t i = threadIdx.x >> wide; i < args.blocks; i += kSortThreads >> wide) {
                const uint32_t b = i + blockIdx.x < args.blocks ? i + blockIdx.x : i + blockIdx.x - args.blocks;   // (each block from another one on: an L2's channels share the work)
                const uint32_t c = args.part[(size_t)b * args.experts + e];
                all += c;
                some += b < blockIdx.x ? c : 0u;
            }
        }
        totals[threadIdx.x] = all;
        before[threadIdx.x] = some;
    } else if (args.blocks > 1u) {
        totals[threadIdx.x] = before[threadIdx.x] = 0;
        __syncthreads();
        const uint32_t from = blockIdx.x * args.perBlock, to = from + args.perBlock;   // (of few rows)
        count_others<I>(args, before, 0u, from);
        count_others<I>(args, totals, to, args.rows);
    }
    count_rows<I, MOST>(args, count, begin, end, expert);
    if (threadIdx.x < args.experts) {
        if (args.part != nullptr) {
            for (uint32_t i = threadIdx.x; i < kSortThreads; i += 1u << wide) {
                n += totals[i];
                those += before[i];
            }
        } else {
            if (args.blocks > 1u) {
                those = before[threadIdx.x];
                n = those + totals[threadIdx.x];
            }
#pragma unroll
            for (uint32_t w = 0; w < kSortWaves; ++w) n += count[w][threadIdx.x];
        }
    }
    // ---- where an expert's rows begin
    uint32_t upTo = wave_prefix(n), past = wave_prefix(those);
    if (lane == 63u) sums[0][wave] = upTo, sums[1][wave] = past;
    __syncthreads();
    uint32_t every = 0;
    past = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) {
        upTo += w < wave ? sums[0][w] : 0u;
        every += sums[0][w];
        past += sums[1][w];
    }
    if (blockIdx.x == 0 && threadIdx.x < args.experts) args.ends[threadIdx.x] = (int32_t)upTo;
    // ---- where a wave's first row of each expert goes (behind the last expert's: the rows of none, of which as many are before this block as its other rows leave)
    auto spread = [&](uint32_t e, uint32_t at) {
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = count[w][e];
            count[w][e] = at;
            at += c;
        }
    };
    if (threadIdx.x < args.experts) spread(threadIdx.x, upTo - n + those);
    if (threadIdx.x == kSortThreads - 1u) {
        const uint64_t from = (uint64_t)blockIdx.x * args.perBlock;
        spread(args.experts, every + (uint32_t)(from < args.rows ? from : args.rows) - past);
    }
    __syncthreads();
    const uint32_t bits = 32u - (uint32_t)__builtin_clz(args.experts);
    for (uint32_t first = begin; first < end; first += 64u * kSortTurns) {
        if (end - begin > 64u * kSortTurns) load_experts<I>(args, first, end, expert);
#pragma unroll
        for (uint32_t i = 0; i < kSortTurns; ++i) {
            const uint32_t row = first + 64u * i + lane, e = expert[i];
            const bool on = e != kNoRow;
            uint64_t same = __ballot(on);
            if (same == 0) break;
            for (uint32_t b = 0; b < bits; ++b) {
                const bool set = (e >> b) & 1u;
                const uint64_t those_set = __ballot(set);
                same &= set ? those_set : ~those_set;
            }
            const uint32_t rank = (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1ull));
            if (on) {
                volatile uint32_t *const next = &count[wave][e];   // (a wave's own: its accesses stay in order)
                const uint32_t at = *next + rank;
                if (rank == 0) *next = at + (uint32_t)__builtin_popcountll(same);
                args.back[row] = (int32_t)at;
                if (at < args.rows) args.order[at] = (int32_t)row;   // (it is, unless the choices change meanwhile)
            }
        }
    }
}

// Blocks of a sort.  Up to 32768 rows of 1024 each, in one launch, every block counting the others' rows itself (us, one launch / two, 128 experts: 4096 rows 5.0 / 7.0, 16384 6.0 /
// 7.5, 32768 7.5 / 7.9, 49152 9.1 / 8.3; half as many rows where few experts share LDS's atomics, 16 of them: 16384 6.5 / 7.1, 32768 9.0 / 7.4, 32 of them: 32768 7.5 / 7.4; and a second launch is 3 us on the
// host); then of 1024 rows or more, whose counts come from a first launch and are summed by every block (blocks of 1024 / 2048 / 4096: 131072 rows to 128
// experts 10.5 / 9.6 / 10.2, to 1024 31 / 21 / 19).
constexpr uint32_t kSortRecount = 32768, kSortBlock = 1024, kMostSortBlocks = 256;

bool sort_counts_first(uint32_t rows, uint32_t experts) { return rows > (experts < 32 ? kSortRecount / 2 : kSortRecount); }

uint32_t sort_blocks(uint32_t rows, uint32_t experts)
{
    const uint64_t counts = (uint64_t)rows * experts;
    const uint32_t block = kSortBlock << (!sort_counts_first(rows, experts) ? 0 : counts > (1u << 25) ? 2 : counts > (1u << 22) ? 1 : 0);
    const uint32_t blocks = rows / block + (rows % block != 0);
    return rows == 0 ? 1 : blocks < kMostSortBlocks ? blocks : kMostSortBlocks;
}

template <typename I, uint32_t MOST>
static int launch_sort_type(const SortArgs &a, hipStream_t stream)
{
    if (a.part != nullptr) {
        hipLaunchKernelGGL((count_by_expert_kernel<I, MOST>), dim3(a.blocks), dim3(kSortThreads), 0, stream, a);
        const int e = (int)hipGetLastError();
        if (e) return e;
    }
    hipLaunchKernelGGL((sort_by_expert_kernel<I, MOST>), dim3(a.blocks), dim3(kSortThreads), 0, stream, a);
    return (int)hipGetLastError();
}

int launch_sort(uint32_t choiceBits, SortArgs a, void *stream)
{
    a.blocks = sort_blocks(a.rows, a.experts);
    const uint64_t each = (a.rows + (uint64_t)a.blocks - 1u) / a.blocks;
    a.perBlock = (uint32_t)((each + kSortBlock - 1u) / kSortBlock * kSortBlock);
    if (!sort_counts_first(a.rows, a.experts)) a.part = nullptr;
    if (choiceBits == 32) return a.experts <= 256 ? launch_sort_type<int32_t, 256>(a, (hipStream_t)stream) : launch_sort_type<int32_t, 1024>(a, (hipStream_t)stream);
    return a.experts <= 256 ? launch_sort_type<int64_t, 256>(a, (hipStream_t)stream) : launch_sort_type<int64_t, 1024>(a, (hipStream_t)stream);
}

}  // namespace catcoc
