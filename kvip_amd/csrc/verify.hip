// Verification of drafted tokens against the target's probabilities (kvip_hip_draft.h).
//
// The walk needs one probability per drafted token, p(its parent's row, the token), so it is decided
// before any row is read whole; then one row per request is (two after a refused child of a drawn
// chain): its weights' sum, and the place where the running sum passes the drawn share.
// What bounds it: reading those rows. They are split over workgroups of 4096 weights. Each repeats the
// walk (one wave, a lane per token: one gather, then register work) instead of a launch before it,
// sums its weights in 64 bits and counts itself on the request's ticket; the last one adds up the
// sums in order, finds the part that holds the place and goes through it again (from the cache).
// Where a refusal leaves no weight, that last workgroup goes through the whole row alone (rare).
// 64 chains of 5 tokens over 131072 fp32 weights take 27-28 us, of which reading the 67 MB is 13; the rest is the
// walk before it (four dependent loads) and the last workgroup's round after it. 16 trees over 32000: 11.3 us.
// The sums cross workgroups as atomics of agent scope, which are carried out where all XCDs see them: an
// exchange whose answer is waited for before the ticket is drawn, and loads after the last ticket. (A
// release and an acquire around the ticket write back and invalidate the XCD's L2 in every workgroup: 72 us
// instead of 27, with the tickets side by side.)
#include "kvip_device.h"
#include "kvip_hip_draft.h"

namespace kvip {
namespace {

constexpr int kPart = 4096;                                // weights per workgroup
constexpr int kMaxParts = (1 << 20) / kPart;
constexpr int kTicketWords = 32;                          // a line per ticket: atomics on one line queue up, 12 ns each

template <typename T> struct Weights;  // 16 bytes of them, at any element address
template <> struct Weights<float> { typedef float vec __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Weights<__bf16> { typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Weights<_Float16> { typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2))); };

// The value of lane `lane` (uniform), without an LDS round trip.
KVIP_DEVICE double lane_double(double v, int lane) {
    return __builtin_bit_cast(double, readlane64(__builtin_bit_cast(int64_t, v), lane));
}

// v of the lane that a DPP row shift names, 0 past the row of 16 lanes.
template <int CTRL>
KVIP_DEVICE double dpp_double(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp_row<CTRL>(static_cast<uint32_t>(bits)), hi = dpp_row<CTRL>(static_cast<uint32_t>(bits >> 32));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Inclusive running sum over the lanes; lane 63 has the whole.
KVIP_DEVICE double wave_running(double v) {
    v += dpp_double<0x111>(v);  // row_shr:1
    v += dpp_double<0x112>(v);
    v += dpp_double<0x114>(v);
    v += dpp_double<0x118>(v);
    const double r0 = lane_double(v, 15), r1 = r0 + lane_double(v, 31), r2 = r1 + lane_double(v, 47);
    const int row = lane_id() >> 4;
    return v + (row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

struct Walk {
    int end;                              // row (within the request) where the walk ends
    int kept;                             // its rows
    int residual;                         // weights are max(probs - draft_probs, 0)
    int excluded;                         // tokens whose weight is 0
    int last;                             // the last chosen child with a weight where the walk ends, -1: none
    int tokens[KVIP_DRAFT_MAX_NODES];
};

// The walk of request b, by one wave. `write`: also its path, and the tokens taken.
template <typename T>
KVIP_DEVICE void walk_request(const KvipVerifyArgs& p, int b, int begin, int n, bool write, Walk* w) {
    const int lane = lane_id();
    const T* probs = static_cast<const T*>(p.probs);
    const T* draft = static_cast<const T*>(p.draft_probs);
    const bool live = lane < n;
    const int64_t token = live ? p.tokens[begin + lane] : -1;
    const bool named = token >= 0 && token < p.vocab;
    int up = !live || lane == 0 ? -1 : p.parents != nullptr ? p.parents[begin + lane] : lane - 1;
    uint32_t err = live && lane > 0 && !named ? KVIP_STATUS_BAD_TOKEN : 0u;
    if (up < -1 || up >= lane) {
        if (live && lane > 0) err |= KVIP_STATUS_BAD_TREE;
        up = -1;
    }
    const bool child = up >= 0 && named;
    double mine = 0.0, drawn = 0.0;
    if (child) {
        mine = static_cast<double>(static_cast<float>(probs[(begin + up) * p.probs_stride + token]));
        if (draft != nullptr) drawn = static_cast<double>(static_cast<float>(draft[(begin + up) * p.draft_stride + token]));
    }
    if (!(mine > 0.0)) mine = 0.0;
    const double uniform = live ? static_cast<double>(p.uniforms[begin + lane]) : 0.0;
    int at = 0, kept = 1, residual = 0;
    int place = lane == 0 ? 0 : -1;  // lane i: row of the walk's i-th token
    unsigned long long tried;
    int last = -1;
    for (;;) {  // at most n rounds: a child comes after its parent
        tried = __ballot(child && up == at);
        last = -1;
        const double u = lane_double(uniform, at);
        int next = -1;
        if (draft != nullptr) {
            const int c = at + 1;
            if (tried != 0) {
                const double q = lane_double(drawn, c), t = lane_double(mine, c);
                if (u * q < t) next = c;
            }
            // A token outside the vocabulary is refused too.
            if (next < 0) residual = c < n;
        } else {
            double low = 0.0;
            unsigned long long left = tried;
            while (left != 0) {
                const int c = __ffsll(left) - 1;
                const int64_t name = __builtin_amdgcn_readlane(static_cast<int>(token), c);  // named: below 2^20
                left &= ~__ballot(child && up == at && token == name);  // named again: nothing left
                const double weight = lane_double(mine, c), high = low + weight;
                if (low <= u && u < high) {
                    next = c;
                    break;
                }
                if (weight > 0.0) last = static_cast<int>(name);
                low = high;
            }
        }
        if (next < 0) break;
        at = next;
        if (lane == kept) place = at;
        ++kept;
    }
    if (lane == 0) {
        w->end = at;
        w->kept = kept;
        w->residual = residual;
        w->excluded = draft != nullptr ? 0 : __popcll(tried);
        w->last = last;
    }
    if (draft == nullptr && (tried >> lane & 1)) {
        w->tokens[__popcll(tried & ((1ull << lane) - 1))] = static_cast<int>(token);
    }
    if (!write) return;
    report(p.status, err);
    const int64_t following = __shfl(static_cast<int>(token), max(__shfl(place, min(lane + 1, 63)), 0));
    if (lane < p.max_nodes) {
        p.path[static_cast<int64_t>(b) * p.max_nodes + lane] = place;
        if (lane + 1 != kept) {  // the drawn token comes from the request's last workgroup
            p.out_tokens[static_cast<int64_t>(b) * p.max_nodes + lane] = lane + 1 < kept ? following : -1;
        }
    }
    if (lane == 0) p.kept[b] = kept;
}

// THREADS: 512 where all workgroups are on the card at once with that (a thread's weights are added up one after
// the other: 16 trees over 32000 take 11.1 us, 11.8 with 256), else 256 (64 chains over 131072: 27.0, 28.1 with 512).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void verify_kernel(const KvipVerifyArgs p) {
    constexpr int kPerLane = kPart / THREADS;  // weights per thread
    typedef typename Weights<T>::vec V;
    constexpr int kLoad = 16 / sizeof(T);
    __shared__ Walk s_walk;
    __shared__ double s_wave[THREADS / 64], s_before, s_left;
    __shared__ int s_last, s_part, s_found, s_near, s_count, s_gone[KVIP_DRAFT_MAX_NODES];
    const int part = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int first = p.cu_seqlens[b], behind = p.cu_seqlens[b + 1];
    const int begin = min(max(first, 0), p.max_tokens), end = min(max(behind, begin), p.max_tokens);
    const bool refused = p.steps != nullptr && p.steps[b] <= 0;
    const int all = refused ? 0 : end - begin;
    const int n = min(all, p.max_nodes);
    if (part == 0 && tid == 0 && (all > n || begin != first || end != behind)) report(p.status, KVIP_STATUS_BAD_LENGTH);
    if (n == 0) {  // uniform over the request's workgroups: its ticket is not used
        if (part == 0 && tid < p.max_nodes) {
            p.path[static_cast<int64_t>(b) * p.max_nodes + tid] = -1;
            p.out_tokens[static_cast<int64_t>(b) * p.max_nodes + tid] = -1;
            if (tid == 0) p.kept[b] = 0;
        }
        return;
    }
    if (wave == 0) walk_request<T>(p, b, begin, n, part == 0, &s_walk);
    if (tid == 0) s_count = 0;
    __syncthreads();
    const int64_t row = begin + s_walk.end;
    const T* probs = static_cast<const T*>(p.probs) + row * p.probs_stride;
    const T* draft = s_walk.residual ? static_cast<const T*>(p.draft_probs) + row * p.draft_stride : nullptr;

    // The weights [at, at + kLoad) of the row, in 64 bits: exact.
    auto weights = [&](int at, double* out) {
        V a{}, d{};
        if (at + kLoad <= p.vocab) {
            a = *reinterpret_cast<const V*>(probs + at);
            if (draft != nullptr) d = *reinterpret_cast<const V*>(draft + at);
        } else {
#pragma unroll
            for (int e = 0; e < kLoad; ++e) {
                if (at + e < p.vocab) {
                    a[e] = probs[at + e];
                    if (draft != nullptr) d[e] = draft[at + e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kLoad; ++e) {
            const double x = static_cast<double>(static_cast<float>(a[e])) - static_cast<double>(static_cast<float>(d[e]));
            out[e] = x > 0.0 ? x : 0.0;  // also a NaN
        }
    };
    auto exclude = [&](int at, double* x, int count, const int* gone) {
        for (int k = 0; k < count; ++k) {
#pragma unroll
            for (int e = 0; e < kLoad; ++e) {
                if (gone[k] == at + e) x[e] = 0.0;
            }
        }
    };
    // Of the excluded tokens, those of part `which` (few or none).
    auto gather_gone = [&](int which) {
        if (tid < s_walk.excluded) {
            const int t = s_walk.tokens[tid];
            if (t / kPart == which) s_gone[atomicAdd(&s_count, 1)] = t;
        }
        __syncthreads();
    };
    gather_gone(part);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPerLane / kLoad; ++j) {
        const int at = part * kPart + (j * THREADS + tid) * kLoad;
        double x[kLoad];
        weights(at, x);
        exclude(at, x, s_count, s_gone);
#pragma unroll
        for (int e = 0; e < kLoad; ++e) sum += x[e];
    }
    sum = wave_running(sum);
    if (lane == 63) s_wave[wave] = sum;
    __syncthreads();
    // The tickets first, at the same place for every shape: they are 0 between calls, whatever the sums behind hold.
    uint32_t* ticket = static_cast<uint32_t*>(p.workspace) + b * kTicketWords;
    double* sums = reinterpret_cast<double*>(static_cast<uint32_t*>(p.workspace) + KVIP_DRAFT_MAX_BATCH * kTicketWords) +
                   static_cast<int64_t>(b) * gridDim.x;
    if (tid == 0) {
        double whole = 0.0;
#pragma unroll
        for (int k = 0; k < THREADS / 64; ++k) whole += s_wave[k];
        uint64_t before = __hip_atomic_exchange(reinterpret_cast<uint64_t*>(sums + part), __builtin_bit_cast(uint64_t, whole),
                                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" : "+v"(before));  // the exchange has been done
        s_last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        if (s_last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;

    // The part in which the running sum passes the share, and the sum before it: one part per thread
    // in order.
    static_assert(kMaxParts <= THREADS, "a part per thread");
    double mine = tid < static_cast<int>(gridDim.x)
                      ? __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<uint64_t*>(sums + tid),
                                                                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) : 0.0;
    // Runs a block-wide inclusive sum of v; returns it, and the whole to *total.
    auto running = [&](double v, double* total) {
        const double in_wave = wave_running(v);
        __syncthreads();
        if (lane == 63) s_wave[wave] = in_wave;
        __syncthreads();
        double before = 0.0, whole = 0.0;
#pragma unroll
        for (int k = 0; k < THREADS / 64; ++k) {
            before += k < wave ? s_wave[k] : 0.0;
            whole += s_wave[k];
        }
        *total = whole;
        return before + in_wave;
    };
    double whole;
    double upto = running(mine, &whole);
    if (whole == 0.0 && draft != nullptr) {
        // A target that is nowhere above its draft (the refused token was a rounding step below): drawn from itself,
        // by this workgroup alone, as it is rare.
        draft = nullptr;
        for (int k = 0; k < static_cast<int>(gridDim.x); ++k) {
            double of_part = 0.0, part_sum;
#pragma unroll
            for (int j = 0; j < kPerLane / kLoad; ++j) {
                double x[kLoad];
                weights(k * kPart + (j * THREADS + tid) * kLoad, x);
#pragma unroll
                for (int e = 0; e < kLoad; ++e) of_part += x[e];
            }
            running(of_part, &part_sum);
            if (tid == k) mine = part_sum;
        }
        upto = running(mine, &whole);
    }
    const double target = static_cast<double>(p.final_uniforms[b]) * whole;
    if (tid == 0) {
        s_part = kMaxParts;
        s_near = -1;
        s_found = 1 << 30;
        s_count = 0;
    }
    __syncthreads();
    const bool drawable = whole > 0.0 && whole <= 1.7976931348623157e308;
    if (mine > 0.0) {
        if (upto > target) atomicMin(&s_part, tid);
        atomicMax(&s_near, tid);  // a share of 1 or one lost to rounding: the last part with a weight
    }
    __syncthreads();
    const int chosen = s_part < kMaxParts ? s_part : s_near;
    if (drawable && tid == chosen) {
        s_before = upto - mine;
        s_left = target;
    }
    __syncthreads();
    int64_t drawn = -1;
    if (drawable) {
        gather_gone(chosen);
        if (tid == 0) s_near = -1;
        // In order: kPerLane weights in a row per thread.
        const int at = chosen * kPart + tid * kPerLane;
        double x[kPerLane], own = 0.0;
#pragma unroll
        for (int j = 0; j < kPerLane / kLoad; ++j) {
            weights(at + j * kLoad, x + j * kLoad);
            exclude(at + j * kLoad, x + j * kLoad, s_count, s_gone);
        }
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) own += x[e];
        double unused;
        double sum_to = running(own, &unused) - own + s_before;
        int found = 1 << 30, last = -1;
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) {
            sum_to += x[e];
            if (x[e] > 0.0) {
                if (sum_to > s_left && found == 1 << 30) found = at + e;
                last = at + e;
            }
        }
        if (found < 1 << 30) atomicMin(&s_found, found);
        if (last >= 0) atomicMax(&s_near, last);
        __syncthreads();
        drawn = s_found < 1 << 30 ? s_found : s_near;
    } else if (whole == 0.0) {
        drawn = s_walk.last;  // children that are the whole target, whose probabilities fall short of 1 by a rounding
    }
    if (tid == 0) {
        if (drawn < 0) report(p.status, KVIP_STATUS_BAD_PROBS);
        p.out_tokens[static_cast<int64_t>(b) * p.max_nodes + s_walk.kept - 1] = drawn;
    }
}

int verify_parts(int vocab) { return (vocab + kPart - 1) / kPart; }

constexpr int kCardWaves = 256 * 32;  // waves that the card holds

template <typename T>
void launch_verify(const KvipVerifyArgs& a, hipStream_t s) {
    const dim3 grid(verify_parts(a.vocab), a.batch);
    if (static_cast<int64_t>(grid.x) * grid.y * (512 / 64) <= kCardWaves) {
        hipLaunchKernelGGL((verify_kernel<T, 512>), grid, dim3(512), 0, s, a);
    } else {
        hipLaunchKernelGGL((verify_kernel<T, 256>), grid, dim3(256), 0, s, a);
    }
}

}  // namespace
}  // namespace kvip

extern "C" uint64_t kvip_hip_verify_drafts_workspace_bytes(int32_t batch, int32_t vocab) {
    if (batch < 1 || vocab < 1) return 0;
    return static_cast<uint64_t>(KVIP_DRAFT_MAX_BATCH) * kvip::kTicketWords * sizeof(uint32_t) +
           static_cast<uint64_t>(batch) * kvip::verify_parts(vocab) * sizeof(double);
}

extern "C" uint32_t kvip_hip_verify_drafts(const KvipVerifyArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    const bool ok = a->probs && a->tokens && a->cu_seqlens && a->uniforms && a->final_uniforms && a->out_tokens && a->kept &&
                    a->path && a->workspace && (reinterpret_cast<uintptr_t>(a->workspace) & 7u) == 0 &&
                    (a->draft_probs == nullptr || a->parents == nullptr) && a->batch >= 1 &&
                    a->batch <= KVIP_DRAFT_MAX_BATCH && a->max_nodes >= 1 && a->max_nodes <= KVIP_DRAFT_MAX_NODES &&
                    a->max_tokens >= 1 && a->max_tokens <= KVIP_DRAFT_MAX_TOKENS && a->vocab >= 1 && a->vocab <= (1 << 20) &&
                    a->probs_stride >= a->vocab && (a->draft_probs == nullptr || a->draft_stride >= a->vocab) &&
                    (a->dtype == KVIP_DTYPE_FP32 || a->dtype == KVIP_DTYPE_BF16 || a->dtype == KVIP_DTYPE_FP16);
    if (!ok) return KVIP_ERR_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    switch (a->dtype) {
        case KVIP_DTYPE_FP32: kvip::launch_verify<float>(*a, s); break;
        case KVIP_DTYPE_BF16: kvip::launch_verify<__bf16>(*a, s); break;
        default: kvip::launch_verify<_Float16>(*a, s); break;
    }
    return static_cast<uint32_t>(hipGetLastError());
}
