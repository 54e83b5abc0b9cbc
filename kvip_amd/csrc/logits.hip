// Logits to probabilities (penalties, biases, grammar masks, temperature) and the histories that the penalties
// read (kvip_hip_prompt.h).
//
// Nearly all of a row is alike: a logit, a bit whether the request holds the token, for those it holds a count, a
// bit whether the grammar allows it. Only the row's drafted ancestors and the request's biases (some hundred
// tokens of a vocabulary) need more, and each of these is worked out by one thread on its own: a bit in LDS takes
// the token out of the dense pass, the thread puts it back. So lists of any length cost the dense pass nothing. A
// token named several times has a second bit: the thread of the first entry that names it has it, and its wave goes through the
// list together, so that neither its sum nor the order of the row's depends on which thread comes first.
//
// A row is read twice: for its maximum and sum, a part of the vocabulary per workgroup, then, in a second launch, for its
// probabilities, each workgroup putting the parts' statistics together for itself. (A row that is one part takes one launch.) The
// first reading is the running maximum and sum of a softmax, per thread, without a branch; NaN and infinities are
// looked for only where the sum is no number.
//
// What bounds it. 320 rows of 131072 bf16 logits: 37 + 52 us in turn over one input (some of which the last cache keeps; 104 a
// pass over others). The second launch moves 252 MB at 4.8 TB/s; the first is bound by vector instructions (28 per token and lane,
// of which 10 are the penalties, worked out for a whole wave wherever one of its 512 tokens is held) and by its last round
// of workgroups. 176 constrained rows of 32000 with 64 biases 11 + 14 us, one row of 131072 fp32 logits 5.3 + 6.1 us: chains of
// latencies (request, its numbers, lists, bits, counts). 8 rows of 30000 with 4096 biases take 18.5 us, 26 with one token
// named twice, 580 with all of them.
// A token takes its bias from the entry that names it; the list is gone through only where several entries name one.
// Dropped after measuring: held tokens taken out of the dense pass and worked out from a list (39 + 87 us; the scattered stores
// cost more than the penalties), biases staged in LDS (20 % more for the constrained rows), 256 or 1024
// threads per workgroup (-2 %, +25 %).
#include "kvip_hip_prompt.h"
#include "lane_groups.h"

namespace kvip {
namespace {

constexpr int kLgThreads = 512;
constexpr int kLgWaves = kLgThreads / 64;
constexpr int kLgVec = 8;                      // tokens of a thread at a time: a byte of the bit masks
constexpr int kLgRun = kLgThreads * kLgVec;
constexpr int kLgListed = 4;                   // entries of a lane looked at together
constexpr int kLgMaxPart = 1 << 17;            // tokens of a workgroup (twice 16 KB of bits)
constexpr float kLgLog2e = 1.44269504088896341f;
constexpr float kLgLargest = 3.402823466e38f;

template <typename T> struct Logits { typedef T vec __attribute__((ext_vector_type(kLgVec), aligned(sizeof(T)))); };
typedef int LogitCounts __attribute__((ext_vector_type(kLgVec), aligned(4)));

struct LogitStat {
    float m, l;  // largest x, sum of exp((x - m) / temperature)
    int first;   // first token of the largest x
    int reserved;
};

struct LogitRow {
    float repetition, inverse, presence, frequency;
    float c;      // log2(e) / temperature
    bool greedy;
    bool plain;   // c is an ordinary number, so that exp2((x - m) c) needs no care but for an m of infinity
};

// All bits where bit i of x is set, else none; and a where `on` has bits, b where it has none.
KVIP_DEVICE uint32_t bit_mask(uint32_t x, int i) { return static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(x), i, 1)); }
KVIP_DEVICE uint32_t pick(uint32_t on, uint32_t a, uint32_t b) { return (a & on) | (b & ~on); }

KVIP_DEVICE float weight_of(float x, float m, const LogitRow& r) {
    if (r.plain && m < INFINITY) return __builtin_amdgcn_exp2f((x - m) * r.c);
    // Beside an infinite m nothing has weight but its equals, at any temperature.
    return x == m ? 1.f : x == -INFINITY || m == INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaxf(x - m, -kLgLargest) * r.c);
}

// All threads' statistics put together, in every thread: largest first, then sums and places under it.
KVIP_DEVICE void merge_block(LogitStat& a, LogitStat* s_stats, const LogitRow& r) {
    const int w = threadIdx.x >> 6;
    const float most = group_max<64>(a.m);
    if ((threadIdx.x & 63) == 0) s_stats[w].m = most;
    __syncthreads();
    float all = s_stats[0].m;
#pragma unroll
    for (int i = 1; i < kLgWaves; ++i) all = fmaxf(all, s_stats[i].m);
    const float l = group_sum<64>(a.m == -INFINITY ? 0.f : a.l * weight_of(a.m, all, r));
    int first = a.m == all ? a.first : 0x7FFFFFFF;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) first = min(first, __shfl_xor(first, d));
    if ((threadIdx.x & 63) == 0) {
        s_stats[w].l = l;
        s_stats[w].first = first;
    }
    __syncthreads();
    a = {all, s_stats[0].l, s_stats[0].first, 0};
#pragma unroll
    for (int i = 1; i < kLgWaves; ++i) {
        a.l += s_stats[i].l;
        a.first = min(a.first, s_stats[i].first);
    }
}

// A row's part [begin, end) of the vocabulary.
template <typename T>
struct LogitPart {
    const KvipLogitArgs& p;
    const T* logits;
    const int32_t* counts;    // of the request, or null
    const uint8_t* seen;
    const uint8_t* allowed;   // or null
    const uint32_t* special;  // LDS: tokens that are not the dense pass's
    int begin, end;
    LogitRow row;
    uint32_t err;

    // Eight tokens from v on (a multiple of 8) as they lie in memory, and which of them the grammar allows.
    struct Raw {
        typename Logits<T>::vec x;
        uint32_t may, held;  // held: by the request, where that is known
    };
    KVIP_DEVICE Raw fetch(int v) const {
        Raw raw;
        raw.may = raw.held = 0;
        const int there = min(end - v, kLgVec);
        if (there <= 0) return raw;
        raw.may = (1u << there) - 1;
        if (allowed != nullptr) raw.may &= allowed[v >> 3];
        if (seen != nullptr) raw.held = seen[v >> 3];
        if (there == kLgVec) {
            raw.x = *reinterpret_cast<const typename Logits<T>::vec*>(logits + v);
        } else {
#pragma unroll
            for (int i = 0; i < kLgVec; ++i) raw.x[i] = i < there ? logits[v + i] : static_cast<T>(0.f);
        }
        return raw;
    }

    // x of a held token that the request wrote n times, as exact as 32 bits are: where quotient and difference are 32-bit
    // numbers they come out as these, so that tokens whose x are equal tie. (The quotient by the reciprocal and what that leaves,
    // where it leaves a number.)
    KVIP_DEVICE float penalised(float x, int n) const {
        const float less = n > 0 ? fmaf(row.frequency, static_cast<float>(n), row.presence) : 0.f;
        const float product = x * row.inverse, rest = fmaf(-product, row.repetition, x);
        const float quotient = fabsf(rest) < INFINITY ? fmaf(rest, row.inverse, product) : product;
        return x > 0.f ? quotient - less : fmaf(x, row.repetition, -less);
    }

    // Their x, -infinity for those that are not the dense pass's; CAREFUL: and for NaN, which is noted. Without CAREFUL a
    // quotient is a product with the rounded reciprocal, off by 2^-23 at most, which no probability shows; CAREFUL is the way
    // of rows that look for their largest x alone, where a tie has to be one.
    template <bool CAREFUL>
    KVIP_DEVICE void adjust(int v, Raw raw, float (&x)[kLgVec]) {
#pragma unroll
        for (int i = 0; i < kLgVec; ++i) x[i] = static_cast<float>(raw.x[i]);
        if (special != nullptr) raw.may &= ~(special[(v - begin) >> 5] >> (v & 31));
        const uint32_t held = raw.held & raw.may;
        if (held != 0) {
            LogitCounts n;
            if (end - v >= kLgVec) {
                n = *reinterpret_cast<const LogitCounts*>(counts + v);
            } else {
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) n[i] = v + i < end ? counts[v + i] : 0;
            }
#pragma unroll
            for (int i = 0; i < kLgVec; ++i) {  // a count counts with its bit alone
                const uint32_t on = bit_mask(held, i);
                const int written = n[i] & static_cast<int>(on);
                if constexpr (CAREFUL) {
                    x[i] = __uint_as_float(pick(on, __float_as_uint(penalised(x[i], written)), __float_as_uint(x[i])));
                    asm volatile("" : "+v"(x[i]));  // one after another, for fewer registers
                    continue;
                }
                const float factor = __uint_as_float(pick(on, __float_as_uint(x[i] > 0.f ? row.inverse : row.repetition), 0x3F800000u));
                const float less = fmaf(row.frequency, static_cast<float>(written), row.presence);
                x[i] = fmaf(x[i], factor, written > 0 ? -less : -0.f);
            }
        }
        if (raw.may != 0xFFu) {
#pragma unroll
            for (int i = 0; i < kLgVec; ++i) {
                x[i] = __uint_as_float(pick(bit_mask(raw.may, i), __float_as_uint(x[i]), 0xFF800000u));
            }
        }
        if constexpr (CAREFUL) {
#pragma unroll
            for (int i = 0; i < kLgVec; ++i) {
                if (x[i] == x[i]) continue;
                err |= KVIP_STATUS_BAD_PROBS;
                x[i] = -INFINITY;
            }
        }
    }

    // x of token v, which entry e names (the row's ancestors first, then the request's list), before its mask and, where other
    // entries name it (`again`), before its biases. False where an ancestor before e names it, which has it then.
    KVIP_DEVICE bool named(int v, int b, int e, bool again, const int* way, int ways, float* out) const {
        const int bias = e - ways;
        const float own = bias >= 0 ? p.bias_values[static_cast<int64_t>(b) * p.biases + bias] : 0.f;
        float x = static_cast<float>(logits[v]);
        bool held = seen != nullptr && (seen[v >> 3] >> (v & 7) & 1);
        int n = held ? counts[v] : 0;
        if (again || bias < 0) {
            for (int i = 0; i < ways; ++i) {
                if (way[i] == v && i < e) return false;
                n += way[i] == v;
                held = held || way[i] == v;
            }
        }
        if (held) x = penalised(x, n);
        *out = !again && bias >= 0 ? x + own : x;
        return true;
    }
    // All biases of token v added to x in the list's order, by a whole wave, whose lanes all pass the same. False where an entry
    // of the list before `bias` names it, which has it then.
    KVIP_DEVICE bool add_biases(int v, int b, int bias, float* x) const {
        const int lane = threadIdx.x & 63;
        const int32_t* names = p.bias_tokens + static_cast<int64_t>(b) * p.biases;
        const float* values = p.bias_values + static_cast<int64_t>(b) * p.biases;
        for (int i = 0; i < p.biases; i += 64 * kLgListed) {
            int name[kLgListed];
#pragma unroll
            for (int j = 0; j < kLgListed; ++j) name[j] = i + 64 * j + lane < p.biases ? names[i + 64 * j + lane] : -1;
#pragma unroll
            for (int j = 0; j < kLgListed; ++j) {
                for (uint64_t found = __ballot(name[j] == v); found != 0; found &= found - 1) {
                    const int e = i + 64 * j + __builtin_ctzll(found);
                    if (e < bias) return false;
                    *x += values[e];
                }
            }
        }
        return true;
    }
    KVIP_DEVICE float masked(int v, float x) {
        if (allowed != nullptr && !(allowed[v >> 3] >> (v & 7) & 1)) return -INFINITY;
        if (x == x) return x;
        err |= KVIP_STATUS_BAD_PROBS;
        return -INFINITY;
    }
};

static_assert((63 + KVIP_LOGIT_MAX_BIASES + kLgThreads - 1) / kLgThreads <= 32, "bits of a thread's entries");

enum { kLgStats = 1, kLgWrite = 2 };  // both: a row is one part

template <typename T, typename O, int MODE>
__global__ __launch_bounds__(kLgThreads) void logits_kernel(const KvipLogitArgs p, int parts, int part_size) {
    __shared__ uint32_t s_special[kLgMaxPart / 32], s_twice[kLgMaxPart / 32];
    __shared__ LogitStat s_stats[kLgWaves];
    __shared__ int s_way[64];
    __shared__ int s_ways, s_request;
    const int tid = threadIdx.x, lane = tid & 63;
    const int row = blockIdx.x / parts, part = blockIdx.x % parts;
    const int words = (p.vocab + 31) / 32;
    uint32_t err = 0;
    LogitPart<T> at = {p, static_cast<const T*>(p.logits) + row * p.logits_stride, nullptr, nullptr,
                       p.allowed == nullptr ? nullptr : reinterpret_cast<const uint8_t*>(p.allowed + static_cast<int64_t>(row) * words),
                       nullptr, part * part_size, min((part + 1) * part_size, p.vocab), {}, 0};
    const int first = at.begin + tid * kLgVec;
    // What does not need the request is under way before it is known.
    typename LogitPart<T>::Raw next = at.fetch(first);
    const uint64_t seen_by = p.visible != nullptr ? static_cast<uint64_t>(p.visible[row]) : 0;
    LogitStat* stats = static_cast<LogitStat*>(p.workspace) + static_cast<int64_t>(row) * parts;
    LogitStat stat = {-INFINITY, 0.f, p.vocab, 0};
    if (MODE == kLgWrite && tid < parts) stat = stats[tid];

    if (tid == 0) s_request = p.batch;
    const int listed = (p.visible == nullptr ? 0 : 63) + p.biases;
    if (listed > 0) {
        for (int i = tid; i < (at.end - at.begin + 31) / 32; i += kLgThreads) s_special[i] = s_twice[i] = 0;
    }
    __syncthreads();
    for (int b = tid; b < p.batch; b += kLgThreads) {
        const int from = p.cu_seqlens[b], to = p.cu_seqlens[b + 1];
        if (from <= row && row < to) atomicMin(&s_request, b);
        if (from < 0 || to < from || to > p.max_tokens) err |= KVIP_STATUS_BAD_LENGTH;
    }
    if (blockIdx.x != 0 || (MODE & kLgStats) == 0) err = 0;
    __syncthreads();
    const int b = s_request;
    if (b >= p.batch) {
        report(p.status, err);
        return;
    }
    if (p.seen != nullptr) {
        at.counts = p.counts + static_cast<int64_t>(b) * p.vocab;
        at.seen = reinterpret_cast<const uint8_t*>(p.seen + static_cast<int64_t>(b) * words);
        if (first < at.end) next.held = at.seen[first >> 3];
    }
    const float temperature = p.temperature == nullptr ? 1.f : p.temperature[b];
    at.row.repetition = p.repetition == nullptr ? 1.f : p.repetition[b];
    at.row.inverse = 1.f / at.row.repetition;
    at.row.presence = p.presence == nullptr ? 0.f : p.presence[b];
    at.row.frequency = p.frequency == nullptr ? 0.f : p.frequency[b];
    at.row.greedy = !(temperature > 0.f);
    at.row.c = at.row.greedy ? 1.f : kLgLog2e / temperature;
    at.row.plain = at.row.c > 0.f && at.row.c < INFINITY;

    // The row's ancestors, and which tokens of this part are not the dense pass's.
    uint32_t mine = 0;  // bit k: entry tid + 512 k names a token of this part
    if (listed > 0) {
        if (tid < 64) {
            const int begin = min(max(p.cu_seqlens[b], 0), p.max_tokens), behind = min(max(p.cu_seqlens[b + 1], begin), p.max_tokens);
            bool on = lane > 0 && begin + lane < behind && (seen_by >> lane & 1);
            const int64_t token = on ? p.tokens[begin + lane] : 0;
            if (on && (token < 0 || token >= p.vocab)) {
                err |= KVIP_STATUS_BAD_TOKEN;
                on = false;
            }
            const uint64_t all = __ballot(on);
            if (on) s_way[__popcll(all & ((1ull << lane) - 1))] = static_cast<int>(token);
            if (lane == 0) s_ways = __popcll(all);
        }
        __syncthreads();
        const int ways = s_ways;
        for (int e = tid, k = 0; e < ways + p.biases; e += kLgThreads, ++k) {
            const int v = e < ways ? s_way[e] : p.bias_tokens[static_cast<int64_t>(b) * p.biases + e - ways];
            if (v >= p.vocab) err |= KVIP_STATUS_BAD_TOKEN;
            if (v < at.begin || v >= at.end) continue;
            const uint32_t bit = 1u << (v & 31);
            mine |= 1u << k;
            if (atomicOr(&s_special[(v - at.begin) >> 5], bit) & bit) atomicOr(&s_twice[(v - at.begin) >> 5], bit);
        }
        __syncthreads();
        at.special = s_special;
    }
    // f(x, token) of this thread's tokens.
    auto for_mine = [&](auto f) {
        for (uint32_t rest = mine; __ballot(rest != 0) != 0; rest &= rest - 1) {  // lanes without a token go along
            const int ways = s_ways, e = tid + (__ffs(rest) - 1) * kLgThreads;
            bool have = rest != 0, again = false;
            int v = 0;
            float x = 0.f;
            if (have) {
                v = e < ways ? s_way[e] : p.bias_tokens[static_cast<int64_t>(b) * p.biases + e - ways];
                again = (s_twice[(v - at.begin) >> 5] >> (v & 31) & 1) != 0;
                have = at.named(v, b, e, again, s_way, ways, &x);
            }
            for (uint64_t several = __ballot(have && again); several != 0; several &= several - 1) {
                const int l = __builtin_ctzll(several);
                float sum = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
                const bool first_named = at.add_biases(__builtin_amdgcn_readlane(v, l), b, __builtin_amdgcn_readlane(e, l) - ways, &sum);
                if (lane == l) {
                    x = sum;
                    have = first_named;
                }
            }
            if (have) f(at.masked(v, x), v);
        }
    };

    if constexpr ((MODE & kLgStats) != 0) {
        const bool ordinary = !at.row.greedy && at.row.plain;
        if (ordinary) {
            // The largest so far starts as the lowest number, so that every difference is one. Infinities and NaN come out as
            // a sum that is none.
            float top = -kLgLargest, l = 0.f;
            for (int v = first; v < at.end; v += kLgRun) {
                const auto raw = next;
                next = at.fetch(v + kLgRun);
                float x[kLgVec], most = top;
                at.template adjust<false>(v, raw, x);
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) most = fmaxf(most, x[i]);
                l *= __builtin_amdgcn_exp2f((top - most) * at.row.c);
                top = most;
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) l += __builtin_amdgcn_exp2f((x[i] - top) * at.row.c);
            }
            stat.l = l;
            if (l > 0.f) stat.m = top;
        }
        if (!ordinary || stat.l != stat.l) {
            stat = {-INFINITY, 0.f, p.vocab, 0};
            next = at.fetch(first);
            for (int v = first; v < at.end; v += kLgRun) {
                const auto raw = next;
                next = at.fetch(v + kLgRun);
                float x[kLgVec], most;
                at.template adjust<true>(v, raw, x);
                most = x[0];
#pragma unroll
                for (int i = 1; i < kLgVec; ++i) most = fmaxf(most, x[i]);
                if (most > stat.m) {
                    stat.l *= weight_of(stat.m, most, at.row);
                    stat.m = most;
#pragma unroll
                    for (int i = kLgVec - 1; i >= 0; --i) stat.first = x[i] == most ? v + i : stat.first;
                }
                if (at.row.greedy || stat.m == -INFINITY) continue;
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) stat.l += weight_of(x[i], stat.m, at.row);
            }
        }
        for_mine([&](float x, int v) {
            if (x > stat.m) {
                stat = {x, (stat.m == -INFINITY ? 0.f : stat.l * weight_of(stat.m, x, at.row)) + 1.f, v, 0};
            } else if (x != -INFINITY) {
                stat.l += weight_of(x, stat.m, at.row);
                if (x == stat.m) stat.first = min(stat.first, v);
            }
        });
        merge_block(stat, s_stats, at.row);
        if constexpr (MODE == kLgStats) {
            if (tid == 0) stats[part] = stat;
        } else {
            next = at.fetch(first);
        }
        err |= at.err;
    } else {
        merge_block(stat, s_stats, at.row);
    }
    if constexpr ((MODE & kLgWrite) != 0) {
        if (part == 0 && tid == 0 && stat.m == -INFINITY) err |= KVIP_STATUS_BAD_PROBS;
        const float share = stat.m == -INFINITY ? 0.f : 1.f / stat.l;
        auto prob = [&](float x, int v) {
            if (stat.m == -INFINITY) return 0.f;
            return at.row.greedy ? (v == stat.first ? 1.f : 0.f) : fmaxf(weight_of(x, stat.m, at.row) * share, 0.f);
        };
        const bool fast = !at.row.greedy && at.row.plain && stat.m != -INFINITY && stat.m < INFINITY;
        O* out = static_cast<O*>(p.probs) + row * p.probs_stride;
        for (int v = first; v < at.end; v += kLgRun) {
            const auto raw = next;
            next = at.fetch(v + kLgRun);
            float x[kLgVec];
            at.template adjust<false>(v, raw, x);
            typename Logits<O>::vec y;
            if (fast) {  // a NaN gets 0 from the maximum
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) y[i] = static_cast<O>(fmaxf(__builtin_amdgcn_exp2f((x[i] - stat.m) * at.row.c) * share, 0.f));
            } else {
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) y[i] = static_cast<O>(prob(x[i], v + i));
            }
            if (at.end - v >= kLgVec) {
                *reinterpret_cast<typename Logits<O>::vec*>(out + v) = y;
            } else {
#pragma unroll
                for (int i = 0; i < kLgVec; ++i) {
                    if (v + i < at.end) out[v + i] = y[i];
                }
            }
        }
        if (listed > 0) {
            __syncthreads();  // the dense pass's zeros are in place
            for_mine([&](float x, int v) { out[v] = static_cast<O>(prob(x, v)); });
        }
    }
    report(p.status, err);
}

// A launch has fewer than 2^32 threads.
bool logits_fit(int rows, int parts) { return static_cast<int64_t>(rows) * parts * kLgThreads < (1ll << 32); }

// Parts of a row: enough workgroups for 4 per CU, of whole runs.
void logit_parts(int rows, int vocab, int* parts, int* size) {
    const int64_t runs = (vocab + kLgRun - 1) / kLgRun, most = kLgMaxPart / kLgRun;
    int64_t want = (1024 + rows - 1) / rows;
    want = want < (runs + most - 1) / most ? (runs + most - 1) / most : want > runs ? runs : want;
    const int64_t per = (runs + want - 1) / want;
    *parts = static_cast<int>((runs + per - 1) / per);
    *size = static_cast<int>(per * kLgRun);
}

template <typename T, typename O>
void launch_logits(const KvipLogitArgs& a, hipStream_t s) {
    int parts, size;
    logit_parts(a.max_tokens, a.vocab, &parts, &size);
    const dim3 grid(static_cast<unsigned>(parts) * static_cast<unsigned>(a.max_tokens)), block(kLgThreads);
    if (parts == 1) {
        hipLaunchKernelGGL((logits_kernel<T, O, kLgStats | kLgWrite>), grid, block, 0, s, a, parts, size);
    } else {
        hipLaunchKernelGGL((logits_kernel<T, O, kLgStats>), grid, block, 0, s, a, parts, size);
        hipLaunchKernelGGL((logits_kernel<T, O, kLgWrite>), grid, block, 0, s, a, parts, size);
    }
}

template <typename T>
void launch_logits(const KvipLogitArgs& a, hipStream_t s) {
    switch (a.probs_dtype) {
        case KVIP_DTYPE_BF16: launch_logits<T, __bf16>(a, s); break;
        case KVIP_DTYPE_FP16: launch_logits<T, _Float16>(a, s); break;
        default: launch_logits<T, float>(a, s); break;
    }
}

// A request's counts over one part of the vocabulary, counted in LDS and written whole, so that nothing has to be
// cleared before. 32 requests of 1000-30000 tokens and 131072 counts take 12 us: each part reads all of a request's tokens
// (from the L2 but for the first), eight per thread at a time; parts of half the size took 14.5.
constexpr int kHistThreads = 1024;
constexpr int kHistPart = 1 << 14;  // 64 KB of counts
constexpr int kHistAtOnce = 8;      // tokens of a thread whose loads are issued together

__global__ __launch_bounds__(kHistThreads) void history_load_kernel(const KvipHistoryArgs p, int parts) {
    __shared__ int s_counts[kHistPart];
    __shared__ uint32_t s_seen[kHistPart / 32];
    const int tid = threadIdx.x, i = blockIdx.x / parts, part = blockIdx.x % parts;
    const int request = p.requests[i], first = p.cu_seqlens[i], behind = p.cu_seqlens[i + 1];
    const int most = static_cast<int>(p.max_tokens);
    const int from = min(max(first, 0), most), to = min(max(behind, from), most);
    uint32_t err = from != first || to != behind || request >= p.batch ? KVIP_STATUS_BAD_LENGTH : 0;
    if (part == 0 && tid == 0) report(p.status, err);
    if (request < 0 || request >= p.batch) return;
    const int begin = part * kHistPart, size = min(kHistPart, p.vocab - begin), words = (size + 31) / 32;
    for (int v = tid; v < size; v += kHistThreads) s_counts[v] = 0;
    for (int w = tid; w < words; w += kHistThreads) s_seen[w] = 0;
    __syncthreads();
    const int64_t written = static_cast<int64_t>(from) + max(p.prompt_lens[i], 0);
    err = 0;
    for (int64_t t0 = from + tid; t0 < to; t0 += kHistThreads * kHistAtOnce) {
        int64_t token[kHistAtOnce];
#pragma unroll
        for (int i = 0; i < kHistAtOnce; ++i) {
            const int64_t t = t0 + i * kHistThreads;
            token[i] = t < to ? p.tokens[t] : begin + size;  // no token of this part
        }
#pragma unroll
        for (int i = 0; i < kHistAtOnce; ++i) {
            const int64_t v = token[i], t = t0 + i * kHistThreads;
            if (t < to && (v < 0 || v >= p.vocab)) err = KVIP_STATUS_BAD_TOKEN;
            if (v < begin || v >= begin + size) continue;
            const int at = static_cast<int>(v) - begin;
            atomicOr(&s_seen[at >> 5], 1u << (at & 31));
            if (t >= written) atomicAdd(&s_counts[at], 1);
        }
    }
    if (part == 0) report(p.status, err);
    __syncthreads();
    int32_t* counts = p.counts + static_cast<int64_t>(request) * p.vocab + begin;
    uint32_t* seen = p.seen + static_cast<int64_t>(request) * ((p.vocab + 31) / 32) + begin / 32;
    for (int v = tid; v < size; v += kHistThreads) counts[v] = s_counts[v];
    for (int w = tid; w < words; w += kHistThreads) seen[w] = s_seen[w];
}

__global__ __launch_bounds__(256) void history_append_kernel(const KvipHistoryArgs p) {
    const int at = blockIdx.x * 256 + threadIdx.x, b = at / p.token_stride, i = at % p.token_stride;
    if (b >= p.batch) return;
    const int kept = p.kept[b];
    if (i == 0 && (kept < 0 || kept > p.token_stride)) report(p.status, KVIP_STATUS_BAD_LENGTH);
    if (i >= kept) return;
    const int64_t v = p.tokens[at];
    if (v < 0 || v >= p.vocab) {
        report(p.status, KVIP_STATUS_BAD_TOKEN);
        return;
    }
    atomicAdd(&p.counts[static_cast<int64_t>(b) * p.vocab + v], 1);
    atomicOr(&p.seen[static_cast<int64_t>(b) * ((p.vocab + 31) / 32) + v / 32], 1u << (v % 32));
}

bool valid_history(const KvipHistoryArgs* a) {
    return a != nullptr && a->counts && a->seen && a->tokens && a->batch >= 1 && a->batch <= KVIP_DRAFT_MAX_BATCH &&
           a->vocab >= 1 && a->vocab <= (1 << 20);
}

bool logit_dtype(int32_t t) { return t == KVIP_DTYPE_FP32 || t == KVIP_DTYPE_BF16 || t == KVIP_DTYPE_FP16; }

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_hip_prompt_abi_version(void) { return KVIP_PROMPT_ABI_VERSION; }

extern "C" uint32_t kvip_hip_history_load(const KvipHistoryArgs* a, void* stream) {
    if (!kvip::valid_history(a) || !a->requests || !a->cu_seqlens || !a->prompt_lens || a->count < 1 ||
        a->count > KVIP_DRAFT_MAX_BATCH || a->max_tokens < 0 || a->max_tokens > 0x7FFFFFFF) {
        return KVIP_ERR_INVALID;
    }
    const int parts = (a->vocab + kvip::kHistPart - 1) / kvip::kHistPart;
    hipLaunchKernelGGL(kvip::history_load_kernel, dim3(a->count * parts), dim3(kvip::kHistThreads), 0,
                       static_cast<hipStream_t>(stream), *a, parts);
    return static_cast<uint32_t>(hipGetLastError());
}

extern "C" uint32_t kvip_hip_history_append(const KvipHistoryArgs* a, void* stream) {
    if (!kvip::valid_history(a) || !a->kept || a->token_stride < 1 || a->token_stride > KVIP_DRAFT_MAX_NODES) return KVIP_ERR_INVALID;
    hipLaunchKernelGGL(kvip::history_append_kernel, dim3((a->batch * a->token_stride + 255) / 256), dim3(256), 0,
                       static_cast<hipStream_t>(stream), *a);
    return static_cast<uint32_t>(hipGetLastError());
}

extern "C" uint64_t kvip_hip_process_logits_workspace_bytes(int32_t max_tokens, int32_t vocab) {
    if (max_tokens < 1 || max_tokens > KVIP_DRAFT_MAX_TOKENS || vocab < 1 || vocab > (1 << 20)) return 0;
    int parts, size;
    kvip::logit_parts(max_tokens, vocab, &parts, &size);
    if (!kvip::logits_fit(max_tokens, parts)) return 0;
    return static_cast<uint64_t>(max_tokens) * parts * sizeof(kvip::LogitStat);
}

extern "C" uint32_t kvip_hip_process_logits(const KvipLogitArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    const bool ok = a->logits && a->probs && a->cu_seqlens && a->workspace &&
                    (reinterpret_cast<uintptr_t>(a->workspace) & 15u) == 0 && (a->counts == nullptr) == (a->seen == nullptr) &&
                    (a->tokens == nullptr) == (a->visible == nullptr) && a->biases >= 0 && a->biases <= KVIP_LOGIT_MAX_BIASES &&
                    (a->biases == 0 || (a->bias_tokens && a->bias_values)) && a->batch >= 1 &&
                    a->batch <= KVIP_DRAFT_MAX_BATCH && a->max_tokens >= 1 && a->max_tokens <= KVIP_DRAFT_MAX_TOKENS &&
                    a->vocab >= 1 && a->vocab <= (1 << 20) && a->logits_stride >= a->vocab && a->probs_stride >= a->vocab &&
                    kvip::logit_dtype(a->dtype) && kvip::logit_dtype(a->probs_dtype) &&
                    kvip_hip_process_logits_workspace_bytes(a->max_tokens, a->vocab) != 0;
    if (!ok) return KVIP_ERR_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (a->dtype) {
        case KVIP_DTYPE_BF16: kvip::launch_logits<__bf16>(*a, s); break;
        case KVIP_DTYPE_FP16: kvip::launch_logits<_Float16>(*a, s); break;
        default: kvip::launch_logits<float>(*a, s); break;
    }
    return static_cast<uint32_t>(hipGetLastError());
}
