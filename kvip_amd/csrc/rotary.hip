// Rotary positions of queries and keys, and the rows of the paged KV cache (kvip_hip_draft.h).
//
// Pair i of a token at position t turns by the angle t * f_i. The turns t * f_i / (2 pi) are taken
// in 64 bits and only their fraction goes on: in 32 bits an angle of 10^6 radians would be off by
// 0.06. sin and cos of the fraction are 32-bit (sincospif, within 2 units in the last place), the
// rotation is 32-bit and each feature is rounded once to its type.
//
// What bounds it: memory (each feature read and written once), latency for a step's few tokens. The
// angles cost as much as some 40 features, so a workgroup works them out once for a run of tokens
// into LDS and every head of these tokens takes them from there. 8192 tokens of 64 query
// heads and a key of 128 features take 59 us (4.6 TB/s; a large copy reaches 5.1), a step of 256 tokens 4.
#include "kvip_device.h"
#include "kvip_hip_draft.h"

namespace kvip {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kVec = 8;                 // features per access
constexpr int kMaxRotary = 512;
constexpr int kRunPairs = 1024;         // pairs of a workgroup's run of tokens (8 KB of LDS)

// Eight features as they lie in memory, at any element address (the card takes 16-byte accesses at
// 2- and 4-byte addresses).
template <typename T> struct Feature;
template <> struct Feature<__bf16> { typedef __bf16 vec __attribute__((ext_vector_type(kVec), aligned(2))); };
template <> struct Feature<_Float16> { typedef _Float16 vec __attribute__((ext_vector_type(kVec), aligned(2))); };
template <> struct Feature<float> { typedef float vec __attribute__((ext_vector_type(kVec), aligned(4))); };

KVIP_DEVICE float2 turn_of(int64_t position, double frequency, float magnitude, bool inverse) {
    const double turns = static_cast<double>(position) * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    const float fraction = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.0f * fraction, &s, &c);
    return make_float2(c * magnitude, (inverse ? -s : s) * magnitude);
}

template <typename T>
KVIP_DEVICE void turn_pair(T a, T b, float2 t, T* x, T* y) {
    const float fa = static_cast<float>(a), fb = static_cast<float>(b);
    *x = static_cast<T>(fa * t.x - fb * t.y);
    *y = static_cast<T>(fb * t.x + fa * t.y);
}

template <typename T, bool HALF>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const KvipRotaryArgs p, int run) {
    typedef typename Feature<T>::vec V;
    __shared__ __align__(16) float2 s_turn[kRunPairs];
    const int tid = threadIdx.x, pairs = p.rotary_dim / 2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * run;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(run), p.tokens - first));
    for (int i = tid; i < tokens * pairs; i += kRotaryThreads) {
        s_turn[i] = turn_of(p.positions[first + i / pairs], p.frequencies[i % pairs], p.magnitude, p.inverse != 0);
    }
    __syncthreads();
    // Whole vectors of features where the pairs allow it (interleaved: four pairs each, halves: eight pairs
    // in two), else pair by pair.
    const bool vectors = HALF ? pairs % kVec == 0 : p.rotary_dim % kVec == 0;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        const KvipRotaryTensor& t = p.tensors[k];
        if (t.x == nullptr || t.heads == 0) continue;
        const T* in = static_cast<const T*>(t.x);
        T* out = static_cast<T*>(t.out);
        const bool copy = in != out;
        const int units = vectors ? (HALF ? pairs / kVec : p.rotary_dim / kVec) : pairs;
        const int tail = copy ? t.dim - p.rotary_dim : 0;
        const int tails = (tail + kVec - 1) / kVec;  // vectors behind the turned part
        const int per_head = units + tails;
        const int per_token = t.heads * per_head;
        for (int i = tid; i < tokens * per_token; i += kRotaryThreads) {
            const int token = i / per_token, rest = i % per_token, head = rest / per_head, u = rest % per_head;
            const T* x = in + (first + token) * t.x_token + head * t.x_head;
            T* y = out + (first + token) * t.out_token + head * t.out_head;
            const float2* turn = s_turn + token * pairs;
            if (u >= units) {
                const int at = p.rotary_dim + (u - units) * kVec;
                if (at + kVec <= t.dim) {
                    *reinterpret_cast<V*>(y + at) = *reinterpret_cast<const V*>(x + at);
                } else {
                    for (int e = at; e < t.dim; ++e) y[e] = x[e];
                }
            } else if (!vectors) {
                T a, b;
                const int ia = HALF ? u : 2 * u, ib = HALF ? pairs + u : 2 * u + 1;
                turn_pair(x[ia], x[ib], turn[u], &a, &b);
                y[ia] = a;
                y[ib] = b;
            } else if constexpr (HALF) {
                const V a = *reinterpret_cast<const V*>(x + u * kVec);
                const V b = *reinterpret_cast<const V*>(x + pairs + u * kVec);
                V c, d;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    T ce, de;
                    turn_pair<T>(a[e], b[e], turn[u * kVec + e], &ce, &de);
                    c[e] = ce;
                    d[e] = de;
                }
                *reinterpret_cast<V*>(y + u * kVec) = c;
                *reinterpret_cast<V*>(y + pairs + u * kVec) = d;
            } else {
                const V a = *reinterpret_cast<const V*>(x + u * kVec);
                V c;
#pragma unroll
                for (int e = 0; e < kVec; e += 2) {
                    T ce, de;
                    turn_pair<T>(a[e], a[e + 1], turn[(u * kVec + e) / 2], &ce, &de);
                    c[e] = ce;
                    c[e + 1] = de;
                }
                *reinterpret_cast<V*>(y + u * kVec) = c;
            }
        }
    }
}

// One wave per token: a lane takes 8 latent features (16 lanes share a scale) and one rotary feature. The
// division is exact to the last bit, as the scale that the reader multiplies by is. 20000 tokens take 11 us
// (3.3 TB/s), a step of 256 tokens 3.3. What bounds many tokens is instructions: 287 VALU ones per wave (nine
// exact divisions and the turn among them) hold the SIMDs for 9.8 of the 11 us.
constexpr int kStoreWaves = 4;
constexpr int kLatent = 512;
constexpr int kRope = 64;

// Largest over the 16 lanes of a row, by rotations within it.
KVIP_DEVICE float row16_max(float x) {
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xF, 0xF, true)));  // row_ror:8
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xF, 0xF, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x122, 0xF, 0xF, true)));
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x121, 0xF, 0xF, true)));
}

template <typename T>
__global__ __launch_bounds__(kStoreWaves * 64) void store_rows_kernel(const KvipRowStoreArgs p) {
    typedef typename Feature<T>::vec V;
    const int lane = threadIdx.x & 63;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * kStoreWaves + (threadIdx.x >> 6);
    if (token >= p.tokens) return;
    const int64_t slot = p.slots[token];
    if (slot < 0) return;
    if (slot >= static_cast<int64_t>(p.num_blocks) * kBlockTokens) {
        if (lane == 0) report(p.status, KVIP_STATUS_BAD_TOKEN);
        return;
    }
    const V raw = *reinterpret_cast<const V*>(static_cast<const T*>(p.latent) + token * p.latent_stride + lane * kVec);
    const T* rope = static_cast<const T*>(p.rope) + token * p.rope_stride;
    const bool turned = p.positions != nullptr;
    const int pair = p.half ? lane & 31 : lane >> 1, other = p.half ? lane ^ 32 : lane ^ 1;
    const float mine = static_cast<float>(rope[lane]), partner = static_cast<float>(rope[other]);

    float x[kVec], largest = 0.f;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
        x[e] = static_cast<float>(raw[e]);
        largest = fmaxf(largest, fabsf(x[e]));
    }
    largest = row16_max(largest);
    const float quotient = largest / 448.f;  // 0 for the smallest magnitudes too, below 3.2e-43
    const float scale = quotient > 0.f ? quotient : 1.f;
    int packed[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
        // A scale below the normal range may be off by more than the format has room for: cut to its largest.
        x[e] = x[e] / scale;
        x[e] = x[e] > 448.f ? 448.f : x[e] < -448.f ? -448.f : x[e];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        packed[e] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * e], x[4 * e + 1], packed[e], false);
        packed[e] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * e + 2], x[4 * e + 3], packed[e], true);
    }
    float feature = mine;
    if (turned) {
        const float2 t = turn_of(p.positions[token], p.frequencies[pair], p.magnitude, false);
        const bool second = p.half ? lane >= 32 : (lane & 1) != 0;
        feature = mine * t.x + (second ? partner : -partner) * t.y;
    }
    uint8_t* row = p.kv_cache + slot / kBlockTokens * p.kv_block_stride + slot % kBlockTokens * p.row_stride;
    *reinterpret_cast<int2*>(row + lane * kVec) = make_int2(packed[0], packed[1]);
    reinterpret_cast<__bf16*>(row + kLatent)[lane] = static_cast<__bf16>(feature);
    if ((lane & 15) == 0) reinterpret_cast<float*>(row + kLatent + 2 * kRope)[lane >> 4] = scale;
}

template <typename T>
void launch_rotary(const KvipRotaryArgs& a, int run, int64_t groups, hipStream_t s) {
    if (a.half) {
        hipLaunchKernelGGL((rotary_kernel<T, true>), dim3(static_cast<unsigned>(groups)), dim3(kRotaryThreads), 0, s, a, run);
    } else {
        hipLaunchKernelGGL((rotary_kernel<T, false>), dim3(static_cast<unsigned>(groups)), dim3(kRotaryThreads), 0, s, a, run);
    }
}

// A launch has fewer than 2^32 threads: longer calls are made in runs of tokens.
constexpr int64_t kLaunchTokens = 1 << 22;

bool valid_tensor(const KvipRotaryTensor& t, int rotary_dim) {
    if (t.x == nullptr) return t.out == nullptr;
    return t.out && t.heads >= 1 && t.heads <= 65536 && t.dim >= rotary_dim && t.dim <= 65536;
}

}  // namespace
}  // namespace kvip

extern "C" uint32_t kvip_hip_rotary(const KvipRotaryArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    const bool ok = a->positions && a->frequencies && a->tokens >= 0 && a->tokens <= (1ll << 31) && a->rotary_dim >= 2 &&
                    a->rotary_dim <= kvip::kMaxRotary && a->rotary_dim % 2 == 0 && a->tensors[0].x &&
                    kvip::valid_tensor(a->tensors[0], a->rotary_dim) && kvip::valid_tensor(a->tensors[1], a->rotary_dim) &&
                    (a->dtype == KVIP_DTYPE_BF16 || a->dtype == KVIP_DTYPE_FP16 || a->dtype == KVIP_DTYPE_FP32);
    if (!ok) return KVIP_ERR_INVALID;
    if (a->tokens == 0) return KVIP_OK;
    // Tokens of a workgroup: enough for each thread to have a vector of features, as many as there is
    // LDS for, and few enough that 1024 workgroups (4 per CU) have some.
    int64_t vectors = 0;
    for (const KvipRotaryTensor& t : a->tensors) {
        if (t.x != nullptr) vectors += static_cast<int64_t>(t.heads) * ((t.dim + kvip::kVec - 1) / kvip::kVec);
    }
    const int64_t fill = (kvip::kRotaryThreads + vectors - 1) / vectors, share = (a->tokens + 1023) / 1024;
    const int64_t room = kvip::kRunPairs / (a->rotary_dim / 2);
    const int64_t want = fill < share ? fill : share;
    const int run = static_cast<int>(want < 1 ? 1 : want > room ? room : want);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t size = a->dtype == KVIP_DTYPE_FP32 ? 4 : 2;
    for (int64_t first = 0; first < a->tokens; first += kvip::kLaunchTokens) {
        KvipRotaryArgs part = *a;
        part.positions += first;
        part.tokens = a->tokens - first < kvip::kLaunchTokens ? a->tokens - first : kvip::kLaunchTokens;
        for (KvipRotaryTensor& t : part.tensors) {
            if (t.x == nullptr) continue;
            t.x = static_cast<const char*>(t.x) + first * t.x_token * size;
            t.out = static_cast<char*>(t.out) + first * t.out_token * size;
        }
        const int64_t groups = (part.tokens + run - 1) / run;
        switch (a->dtype) {
            case KVIP_DTYPE_BF16: kvip::launch_rotary<__bf16>(part, run, groups, s); break;
            case KVIP_DTYPE_FP16: kvip::launch_rotary<_Float16>(part, run, groups, s); break;
            default: kvip::launch_rotary<float>(part, run, groups, s); break;
        }
    }
    return static_cast<uint32_t>(hipGetLastError());
}

extern "C" uint32_t kvip_hip_store_rows(const KvipRowStoreArgs* a, void* stream) {
    if (a == nullptr) return KVIP_ERR_INVALID;
    const bool ok = a->latent && a->rope && a->slots && a->kv_cache && (a->positions == nullptr || a->frequencies) &&
                    a->tokens >= 0 && a->tokens <= (1ll << 31) && a->row_stride >= KVIP_KV_ROW_BYTES && a->row_stride % 16 == 0 &&
                    a->kv_block_stride % 16 == 0 &&
                    a->kv_block_stride >= static_cast<int64_t>(kvip::kBlockTokens) * a->row_stride && a->num_blocks >= 1 &&
                    (reinterpret_cast<uintptr_t>(a->kv_cache) & 15u) == 0 &&
                    (a->dtype == KVIP_DTYPE_BF16 || a->dtype == KVIP_DTYPE_FP16 || a->dtype == KVIP_DTYPE_FP32);
    if (!ok) return KVIP_ERR_INVALID;
    if (a->tokens == 0) return KVIP_OK;
    const dim3 block(kvip::kStoreWaves * 64);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t size = a->dtype == KVIP_DTYPE_FP32 ? 4 : 2;
    for (int64_t first = 0; first < a->tokens; first += kvip::kLaunchTokens) {
        KvipRowStoreArgs part = *a;
        part.latent = static_cast<const char*>(a->latent) + first * a->latent_stride * size;
        part.rope = static_cast<const char*>(a->rope) + first * a->rope_stride * size;
        part.slots += first;
        if (part.positions != nullptr) part.positions += first;
        part.tokens = a->tokens - first < kvip::kLaunchTokens ? a->tokens - first : kvip::kLaunchTokens;
        const dim3 grid(static_cast<unsigned>((part.tokens + kvip::kStoreWaves - 1) / kvip::kStoreWaves));
        switch (a->dtype) {
            case KVIP_DTYPE_BF16: hipLaunchKernelGGL(kvip::store_rows_kernel<__bf16>, grid, block, 0, s, part); break;
            case KVIP_DTYPE_FP16: hipLaunchKernelGGL(kvip::store_rows_kernel<_Float16>, grid, block, 0, s, part); break;
            default: hipLaunchKernelGGL(kvip::store_rows_kernel<float>, grid, block, 0, s, part); break;
        }
    }
    return static_cast<uint32_t>(hipGetLastError());
}
