// Norm of every head of queries and keys and its turn by the token's position in one pass, and for the indexer the
// fp8 features and scale of each head, keys into their paged cache (kvip_hip_prompt.h).
//
// A head is held by G lanes (8 features each, as two runs of four, so that both features of a pair are in one lane in
// either layout); its sums and its largest magnitude are taken over those lanes by DPP and lane swaps. Mean and
// variance are two passes over registers, in 32 bits. Heads of other sizes go through LDS, a wave per head.
// A workgroup takes a run of tokens and works their angles out once; a thread holds its features' weights and has the next
// head's features under way. Few tokens' heads go over several workgroups, their keys to one of their own.
//
// What bounds it: memory for many tokens. 4001 tokens of 32 + 8 normed heads of 128 take 15.5 us (5.3 TB/s; a large copy
// reaches 5.1), 8192 tokens of 64 index heads 49 (4.2 TB/s; 177 vector instructions per 512 features hold the SIMDs for
// some 40 of these, 305 with a division for every feature's code took 71). 256 tokens of 64 index heads take 5.5
// us, one token 3.5: angles, features, codes, one after the other.
#include "kvip_hip_prompt.h"
#include "lane_groups.h"
#include "turn.h"

namespace kvip {
namespace {

constexpr int kNrThreads = 256;
constexpr int kNrWaves = kNrThreads / 64;
constexpr int kNrPairs = 1024;  // pairs of a workgroup's run of tokens (8 KB of LDS)
constexpr int kNrLane = 8;      // features of a lane

template <typename T> struct Four { typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

// Scale of a head whose largest magnitude is given, and a feature under it: as in the rows of the KV cache.
KVIP_DEVICE float head_scale(float largest) {
    const float quotient = largest / 448.f;
    return quotient > 0.f ? quotient : 1.f;
}
KVIP_DEVICE float under_scale(float x, float scale) {  // for any scale
    x /= scale;
    return x > 448.f ? 448.f : x < -448.f ? -448.f : x;
}
// Four features' codes. A quotient is the product with the scale's reciprocal and what that leaves over, which is the rounded
// quotient, and at most 448 but for a rounding, which the conversion rounds away. (The product alone is off by two roundings
// and sends features that are half-way between two codes to either.) A scale so small that what is left over would be below the
// normal range, or one that is infinite, takes divisions.
KVIP_DEVICE float by_reciprocal(float x, float scale, float reciprocal) {
    const float product = x * reciprocal;
    return fmaf(fmaf(-product, scale, x), reciprocal, product);
}
KVIP_DEVICE int head_codes(const float (&x)[4], float scale, float reciprocal) {
    int packed = 0;
    if (scale >= 0x1p-100f && scale < INFINITY) {
        packed = __builtin_amdgcn_cvt_pk_fp8_f32(by_reciprocal(x[0], scale, reciprocal), by_reciprocal(x[1], scale, reciprocal), packed, false);
        return __builtin_amdgcn_cvt_pk_fp8_f32(by_reciprocal(x[2], scale, reciprocal), by_reciprocal(x[3], scale, reciprocal), packed, true);
    }
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(under_scale(x[0], scale), under_scale(x[1], scale), packed, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(under_scale(x[2], scale), under_scale(x[3], scale), packed, true);
}

// Where a head of queries or a key goes: false where nowhere.
struct HeadPlace {
    int64_t out, scale;  // elements
};
KVIP_DEVICE bool head_place(const KvipNormRotaryArgs& p, const KvipNormTensor& t, bool paged, int64_t token, int head, HeadPlace* at,
                            uint32_t* err) {
    if (!paged) {
        at->out = token * t.out_token + head * t.out_head;
        at->scale = token * t.heads + head;
        return true;
    }
    const int64_t slot = p.slots[token];
    if (slot >= static_cast<int64_t>(p.num_blocks) * kBlockTokens) *err |= KVIP_STATUS_BAD_TOKEN;
    if (slot < 0 || slot >= static_cast<int64_t>(p.num_blocks) * kBlockTokens) return false;
    at->out = slot / kBlockTokens * t.out_token + slot % kBlockTokens * kIndexDim;
    at->scale = slot / kBlockTokens * t.out_head + slot % kBlockTokens;
    return true;
}

template <typename T, bool HALF, int G, bool QUANT>
__global__ __launch_bounds__(kNrThreads) void norm_rotary_kernel(const KvipNormRotaryArgs p, int run, int slices) {
    typedef typename Four<T>::vec V;
    typedef Four<float>::vec W;
    constexpr int kGroups = kNrThreads / G;
    __shared__ __align__(16) float2 s_turn[kNrPairs];
    const int tid = threadIdx.x, pairs = p.rotary_dim / 2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * run;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(run), p.tokens - first));
    for (int i = tid; i < tokens * pairs; i += kNrThreads) {
        s_turn[i] = fine_turn_of(p.positions[first + i / pairs], p.frequencies[i % pairs], p.magnitude);
    }
    const int j = tid % G;
    const bool live = j * kNrLane < p.dim, turned = j * kNrLane < p.rotary_dim;
    const int at[2] = {HALF && turned ? 4 * j : 8 * j, HALF && turned ? pairs + 4 * j : 8 * j + 4};
    const float share = 1.f / static_cast<float>(p.dim);
    uint32_t err = 0;
    bool ready = false;  // the angles
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        const KvipNormTensor& t = p.tensors[k];
        if (t.x == nullptr) continue;
        // This slice's heads of the run, counted along tokens and heads. Where the queries have several slices, the keys have one
        // of their own.
        if (slices > 1 && (k == 0) == (blockIdx.y == slices)) continue;
        const int slice = k == 0 ? blockIdx.y : 0, step = k == 0 ? kGroups * slices : kGroups;
        const int by_token = step / t.heads, by_head = step % t.heads;
        int token = (tid / G + slice * kGroups) / t.heads, head = (tid / G + slice * kGroups) % t.heads;
        const T* in = static_cast<const T*>(t.x) + first * t.x_token;
        V raw[2] = {};
        auto fetch = [&] {
            if (token >= tokens || !live) return;
            const T* x = in + token * t.x_token + head * t.x_head;
            raw[0] = *reinterpret_cast<const V*>(x + at[0]);
            raw[1] = *reinterpret_cast<const V*>(x + at[1]);
        };
        fetch();
        W weight[2] = {{1.f, 1.f, 1.f, 1.f}, {1.f, 1.f, 1.f, 1.f}}, bias[2] = {};
        if (t.weight != nullptr && live) {
            weight[0] = *reinterpret_cast<const W*>(t.weight + at[0]);
            weight[1] = *reinterpret_cast<const W*>(t.weight + at[1]);
        }
        if (t.bias != nullptr && live) {
            bias[0] = *reinterpret_cast<const W*>(t.bias + at[0]);
            bias[1] = *reinterpret_cast<const W*>(t.bias + at[1]);
        }
        if (!ready) __syncthreads();
        ready = true;
        while (token < tokens) {
            const int token_now = token, head_now = head;
            float x[kNrLane];
#pragma unroll
            for (int i = 0; i < kNrLane; ++i) x[i] = static_cast<float>(raw[i / 4][i % 4]);
            token += by_token;
            head += by_head;
            if (head >= t.heads) {
                head -= t.heads;
                ++token;
            }
            fetch();
            if (t.norm != KVIP_NORM_NONE) {
                float sum = 0.f;
                if (t.norm == KVIP_NORM_LAYER) {
#pragma unroll
                    for (int i = 0; i < kNrLane; ++i) sum += x[i];
                    const float mean = group_sum<G>(live ? sum : 0.f) * share;
#pragma unroll
                    for (int i = 0; i < kNrLane; ++i) x[i] -= mean;
                    sum = 0.f;
                }
#pragma unroll
                for (int i = 0; i < kNrLane; ++i) sum = fmaf(x[i], x[i], sum);
                const float factor = 1.f / sqrtf(group_sum<G>(live ? sum : 0.f) * share + p.epsilon);
#pragma unroll
                for (int i = 0; i < kNrLane; ++i) x[i] = fmaf(x[i] * factor, weight[i / 4][i % 4], bias[i / 4][i % 4]);
            } else if (t.weight != nullptr || t.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < kNrLane; ++i) x[i] = fmaf(x[i], weight[i / 4][i % 4], bias[i / 4][i % 4]);
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 turn = s_turn[token_now * pairs + 4 * j + i];
                    float& a = x[HALF ? i : 2 * i];
                    float& b = x[HALF ? 4 + i : 2 * i + 1];
                    const float c = a * turn.x - b * turn.y;
                    b = b * turn.x + a * turn.y;
                    a = c;
                }
            }
            HeadPlace place;
            if (!head_place(p, t, QUANT && k == 1, first + token_now, head_now, &place, &err) || !live) continue;
            if constexpr (QUANT) {
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < kNrLane; ++i) largest = fmaxf(largest, fabsf(x[i]));
                const float scale = head_scale(group_max<G>(largest)), reciprocal = 1.f / scale;
                uint8_t* out = static_cast<uint8_t*>(t.out) + place.out;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float four[4] = {x[4 * r], x[4 * r + 1], x[4 * r + 2], x[4 * r + 3]};
                    *reinterpret_cast<int*>(out + at[r]) = head_codes(four, scale, reciprocal);
                }
                if (j == 0) t.scales[place.scale] = scale;
            } else {
                T* out = static_cast<T*>(t.out) + place.out;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    V y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = static_cast<T>(x[4 * r + i]);
                    *reinterpret_cast<V*>(out + at[r]) = y;
                }
            }
        }
    }
    report(p.status, err);
}

// Heads whose features do not come in eights: a wave per head, feature lane + 64 i in register i, pairs met in LDS.
template <typename T>
__global__ __launch_bounds__(kNrThreads) void norm_rotary_any_kernel(const KvipNormRotaryArgs p) {
    constexpr int kPer = KVIP_NORM_MAX_DIM / 64;
    __shared__ float s_head[kNrWaves][KVIP_NORM_MAX_DIM];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, pairs = p.rotary_dim / 2;
    const int heads = p.tensors[0].heads + (p.tensors[1].x != nullptr ? p.tensors[1].heads : 0);
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kNrWaves + w;
    const int64_t token = unit / heads;
    if (token >= p.tokens) return;  // the whole wave, which meets no other
    int head = static_cast<int>(unit % heads);
    const int k = head >= p.tensors[0].heads;
    if (k == 1) head -= p.tensors[0].heads;
    const KvipNormTensor& t = p.tensors[k];
    const T* in = static_cast<const T*>(t.x) + token * t.x_token + head * t.x_head;
    const float share = 1.f / static_cast<float>(p.dim);
    float x[kPer], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        x[i] = lane + 64 * i < p.dim ? static_cast<float>(in[lane + 64 * i]) : 0.f;
        sum += x[i];
    }
    float factor = 1.f, mean = 0.f;
    if (t.norm == KVIP_NORM_LAYER) mean = group_sum<64>(sum) * share;
    if (t.norm != KVIP_NORM_NONE) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] -= mean;
            if (lane + 64 * i < p.dim) sum = fmaf(x[i], x[i], sum);
        }
        factor = 1.f / sqrtf(group_sum<64>(sum) * share + p.epsilon);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int f = lane + 64 * i;
        if (f >= p.dim) continue;
        x[i] *= factor;
        if (t.weight != nullptr || t.bias != nullptr) {
            x[i] = fmaf(x[i], t.weight != nullptr ? t.weight[f] : 1.f, t.bias != nullptr ? t.bias[f] : 0.f);
        }
        s_head[w][f] = x[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float largest = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int f = lane + 64 * i;
        if (f >= p.dim) continue;
        if (f < p.rotary_dim) {
            const int pair = p.half ? f % pairs : f / 2;
            const bool second = p.half ? f >= pairs : (f & 1) != 0;
            const float other = s_head[w][p.half ? (second ? f - pairs : f + pairs) : f ^ 1];
            const float2 turn = fine_turn_of(p.positions[token], p.frequencies[pair], p.magnitude);
            x[i] = x[i] * turn.x + (second ? other : -other) * turn.y;
        }
        largest = fmaxf(largest, fabsf(x[i]));
    }
    HeadPlace place;
    uint32_t err = 0;
    const bool there = head_place(p, t, p.quantised != 0 && k == 1, token, head, &place, &err);
    if (lane == 0) report(p.status, err);
    if (!there) return;
    const float scale = p.quantised != 0 ? head_scale(group_max<64>(largest)) : 1.f;
    if (p.quantised != 0 && lane == 0) t.scales[place.scale] = scale;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int f = lane + 64 * i;
        if (f >= p.dim) continue;
        if (p.quantised != 0) {
            const int code = __builtin_amdgcn_cvt_pk_fp8_f32(under_scale(x[i], scale), 0.f, 0, false);
            static_cast<uint8_t*>(t.out)[place.out + f] = static_cast<uint8_t>(code & 0xFF);
        } else {
            static_cast<T*>(t.out)[place.out + f] = static_cast<T>(x[i]);
        }
    }
}

template <typename T, int G, bool QUANT>
void launch_group(const KvipNormRotaryArgs& a, int run, int slices, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>((a.tokens + run - 1) / run), static_cast<unsigned>(slices > 1 && a.tensors[1].x != nullptr ? slices + 1 : slices)), block(kNrThreads);
    if (a.half) {
        hipLaunchKernelGGL((norm_rotary_kernel<T, true, G, QUANT>), grid, block, 0, s, a, run, slices);
    } else {
        hipLaunchKernelGGL((norm_rotary_kernel<T, false, G, QUANT>), grid, block, 0, s, a, run, slices);
    }
}

template <typename T>
void launch_norm_rotary(const KvipNormRotaryArgs& a, hipStream_t s) {
    const int heads = a.tensors[0].heads + (a.tensors[1].x != nullptr ? a.tensors[1].heads : 0);
    if (a.dim % kNrLane != 0 || a.rotary_dim % kNrLane != 0) {
        const int64_t units = a.tokens * heads;
        hipLaunchKernelGGL(norm_rotary_any_kernel<T>, dim3(static_cast<unsigned>((units + kNrWaves - 1) / kNrWaves)), dim3(kNrThreads),
                           0, s, a);
        return;
    }
    // Lanes of a head, and tokens of a workgroup: enough for each group of lanes to have a head of either array, as many as
    // there is LDS for, and few enough that 1024 workgroups (4 per CU) have some. Few tokens' heads go over more workgroups.
    const int lanes = a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : a.dim <= 256 ? 32 : 64;
    const int groups = kNrThreads / lanes;
    const int least = a.tensors[1].x != nullptr && a.tensors[1].heads < a.tensors[0].heads ? a.tensors[1].heads : a.tensors[0].heads;
    const int64_t fill = (groups + least - 1) / least, share = (a.tokens + 1023) / 1024;
    const int64_t room = kNrPairs / (a.rotary_dim / 2), want = fill < share ? fill : share;
    const int run = static_cast<int>(want < 1 ? 1 : want > room ? room : want);
    const int64_t runs = (a.tokens + run - 1) / run, rounds = (static_cast<int64_t>(run) * a.tensors[0].heads + groups - 1) / groups;
    const int64_t spread = 1024 / runs;
    const int slices = static_cast<int>(spread < 1 ? 1 : spread > rounds ? rounds : spread);
    if (a.quantised) launch_group<T, 16, true>(a, run, slices, s);
    else if (lanes == 8) launch_group<T, 8, false>(a, run, slices, s);
    else if (lanes == 16) launch_group<T, 16, false>(a, run, slices, s);
    else if (lanes == 32) launch_group<T, 32, false>(a, run, slices, s);
    else launch_group<T, 64, false>(a, run, slices, s);
}

bool valid_norm(const KvipNormRotaryArgs& a, int k) {
    const KvipNormTensor& t = a.tensors[k];
    if (t.x == nullptr) return k == 1;
    if (!t.out || t.heads < 1 || t.heads > 65536 || t.norm < KVIP_NORM_NONE || t.norm > KVIP_NORM_LAYER) return false;
    if (!a.quantised) return true;
    // A lane stores four bytes at a time.
    if (!t.scales || (reinterpret_cast<uintptr_t>(t.out) & 3u) != 0 || t.out_token % 4 != 0) return false;
    if (k == 0) return t.out_head % 4 == 0;
    return a.slots && t.heads == 1 && a.num_blocks >= 1 && t.out_token >= kBlockTokens * kIndexDim && t.out_head >= kBlockTokens;
}

// A launch has fewer than 2^32 threads: longer calls are made in runs of tokens.
constexpr int64_t kNrLaunchUnits = 1 << 25;

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_hip_norm_rotary(const KvipNormRotaryArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    const bool ok = a->positions && a->frequencies && a->tokens >= 0 && a->tokens <= (1ll << 31) && a->rotary_dim >= 2 &&
                    a->rotary_dim % 2 == 0 && a->rotary_dim <= a->dim && a->dim <= KVIP_NORM_MAX_DIM &&
                    (!a->quantised || a->dim == KVIP_INDEX_DIM) && a->epsilon >= 0.f && a->epsilon - a->epsilon == 0.f &&
                    kvip::valid_norm(*a, 0) && kvip::valid_norm(*a, 1) &&
                    (a->dtype == KVIP_DTYPE_BF16 || a->dtype == KVIP_DTYPE_FP16 || a->dtype == KVIP_DTYPE_FP32);
    if (!ok) return KVIP_ERR_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t size = a->dtype == KVIP_DTYPE_FP32 ? 4 : 2;
    const int64_t heads = a->tensors[0].heads + (a->tensors[1].x != nullptr ? a->tensors[1].heads : 0);
    const int64_t most = heads > kvip::kNrLaunchUnits ? 1 : kvip::kNrLaunchUnits / heads;
    for (int64_t first = 0; first < a->tokens; first += most) {
        KvipNormRotaryArgs part = *a;
        part.positions += first;
        if (part.slots != nullptr) part.slots += first;
        part.tokens = a->tokens - first < most ? a->tokens - first : most;
        for (int k = 0; k < 2; ++k) {
            KvipNormTensor& t = part.tensors[k];
            if (t.x == nullptr) continue;
            t.x = static_cast<const char*>(t.x) + first * t.x_token * size;
            if (a->quantised && k == 1) continue;  // by slots
            t.out = static_cast<char*>(t.out) + first * t.out_token * (a->quantised ? 1 : size);
            if (a->quantised) t.scales += first * t.heads;
        }
        switch (a->dtype) {
            case KVIP_DTYPE_BF16: kvip::launch_norm_rotary<__bf16>(part, s); break;
            case KVIP_DTYPE_FP16: kvip::launch_norm_rotary<_Float16>(part, s); break;
            default: kvip::launch_norm_rotary<float>(part, s); break;
        }
    }
    return static_cast<uint32_t>(hipGetLastError());
}
