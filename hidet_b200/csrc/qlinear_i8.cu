// Entry point of the int8 x int8 product, and the kernel that takes operands of any alignment.
#include "qlinear_i8.h"
#include "qlinear_i8_plan.h"
#include "serving.cuh"

namespace b200q {
namespace {

// A tile of 64 x 64 by 256 threads, four rows and four columns each, four products an instruction; operands pass through shared memory byte by byte, which is
// what takes the time (333 x 4096 x 4096 334 us, 13 where the weight is aligned; one token 128, 5.6).  For rows that are not multiples of 16 bytes and bases that are not aligned.
constexpr int TILE = 64, STEP = 64, PITCH = STEP / 4 + 1;

__global__ void __launch_bounds__(256) i8_any_kernel(const I8Args p) {
    __shared__ int a_tile[TILE * PITCH], w_tile[TILE * PITCH];
    int8_t *a_bytes = reinterpret_cast<int8_t *>(a_tile), *w_bytes = reinterpret_cast<int8_t *>(w_tile);
    const int n_tiles = (p.N + TILE - 1) / TILE;
    const int m0 = (int)(blockIdx.x / n_tiles) * TILE, n0 = (int)(blockIdx.x % n_tiles) * TILE;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    pdl_launch_dependents();
    pdl_wait();
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += STEP) {
#pragma unroll 4
        for (int i = threadIdx.x; i < TILE * STEP; i += 256) {
            const int r = i / STEP, k = i % STEP;
            a_bytes[r * PITCH * 4 + k] = m0 + r < p.M && k0 + k < p.K ? p.a[(int64_t)(m0 + r) * p.K + k0 + k] : (int8_t)0;
            if (p.nk) {
                w_bytes[r * PITCH * 4 + k] = n0 + r < p.N && k0 + k < p.K ? p.w[(int64_t)(n0 + r) * p.K + k0 + k] : (int8_t)0;
            } else {  // neighbours in a row of the weight, the columns
                w_bytes[k * PITCH * 4 + r] = n0 + k < p.N && k0 + r < p.K ? p.w[(int64_t)(k0 + r) * p.N + n0 + k] : (int8_t)0;
            }
        }
        __syncthreads();
#pragma unroll 4
        for (int k = 0; k < STEP / 4; ++k) {
            int a[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = a_tile[(ty * 4 + i) * PITCH + k], w[i] = w_tile[(tx * 4 + i) * PITCH + k];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], w[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
        if (m >= p.M) continue;
        const float a_scale = p.a_scale[m];
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx * 4 + j;
            y[j] = 0.0f;
            if (n >= p.N) continue;
            y[j] = (float)acc[i][j] * i8_scale(p.scale, p.scale_type, n) * a_scale;
            if (p.bias != nullptr) y[j] += i8_value(p.bias, p.out_type, n);
        }
        const int width = p.pairs ? p.N / 2 : p.N, first = p.pairs ? (n0 + tx * 4) / 2 : n0 + tx * 4, count = p.pairs ? 2 : 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= count || first + j >= width) continue;
            float z = p.pairs ? (j < 2 ? silu(y[(2 * j) & 3]) * y[(2 * j + 1) & 3] : 0.0f) : y[j];
            if (p.residual != nullptr) z += i8_value(p.residual, p.out_type, m * p.ldr + first + j);
            i8_store(p.c, p.out_type, (int64_t)m * width + first + j, z);
        }
    }
}

}  // namespace

int launch_i8_any(const I8Args &p, cudaStream_t stream) {
    const int64_t tiles = ceil_div(p.M, TILE) * ceil_div(p.N, TILE);
    if (tiles > 2147483647LL) return set_error(B200Q_UNSUPPORTED, "qlinear_i8_i8: a product of %d x %d", p.M, p.N);
    return launch_after("i8_any_kernel", i8_any_kernel, dim3((unsigned)tiles), 256, 0, 1, stream, p);
}

}  // namespace b200q

extern "C" {

B200Q_API int b200q_qlinear_i8_i8(const void *a, const float *a_scale, const void *wq, const void *scale, void *c, int64_t M, int64_t N, int64_t K, int w_layout,
                                  int scale_type, int out_type, const b200q_epilogue *epilogue, void *stream) {
    using namespace b200q;
    const char *op = "qlinear_i8_i8";
    if (M < 0 || N < 0 || K < 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: negative size M=%lld N=%lld K=%lld", op, (long long)M, (long long)N, (long long)K);
    if (w_layout != B200Q_LAYOUT_KN && w_layout != B200Q_LAYOUT_NK) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown weight layout %d", op, w_layout);
    if (scale_type < B200Q_F16 || scale_type > B200Q_F32) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown type of the scales %d", op, scale_type);
    if (out_type != B200Q_F16 && out_type != B200Q_BF16) return set_error(B200Q_INVALID_ARGUMENT, "%s: results are f16 or bf16, not type %d", op, out_type);
    const b200q_epilogue none = {nullptr, nullptr, 0, B200Q_ACT_NONE};
    const b200q_epilogue &e = epilogue != nullptr ? *epilogue : none;
    if (e.activation != B200Q_ACT_NONE && e.activation != B200Q_ACT_SILU_MUL) return set_error(B200Q_INVALID_ARGUMENT, "%s: unknown activation %d", op, e.activation);
    const bool pairs = e.activation == B200Q_ACT_SILU_MUL;
    if (pairs && N % 2 != 0) return set_error(B200Q_INVALID_ARGUMENT, "%s: the gate / up pairing needs an even N, got %lld", op, (long long)N);
    const int64_t width = pairs ? N / 2 : N;
    if (e.residual != nullptr && e.ldr < width && M > 1) {
        return set_error(B200Q_INVALID_ARGUMENT, "%s: residual rows of %lld elements are shorter than the result's %lld", op, (long long)e.ldr, (long long)width);
    }
    if (M == 0 || N == 0) return B200Q_OK;
    if (K > kMostInner) return set_error(B200Q_UNSUPPORTED, "%s: K=%lld: sums of up to %lld products fit 32 bits", op, (long long)K, (long long)kMostInner);
    if (M > kMostOuter || N > kMostOuter) return set_error(B200Q_UNSUPPORTED, "%s: M=%lld N=%lld: sizes of 2^31-255 and more are not supported", op, (long long)M, (long long)N);
    if (c == nullptr || scale == nullptr || a_scale == nullptr || (K > 0 && (a == nullptr || wq == nullptr))) return set_error(B200Q_INVALID_ARGUMENT, "%s: null pointer argument", op);
    I8Args p = {};
    p.a = static_cast<const int8_t *>(a), p.w = static_cast<const int8_t *>(wq), p.a_scale = a_scale, p.scale = scale, p.bias = e.bias, p.residual = e.residual;
    p.c = c, p.ldr = e.ldr, p.M = (int)M, p.N = (int)N, p.K = (int)K, p.scale_type = scale_type, p.out_type = out_type, p.pairs = pairs;
    p.nk = w_layout == B200Q_LAYOUT_NK;
    p.status = device_status_word();
    p.residual_vec = p.residual != nullptr && aligned_to(p.residual, 16) && (p.ldr % 8 == 0 || M == 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool lines = aligned_to(a, 16) && aligned_to(wq, 16) && aligned_to(c, 16) && K > 0 && K % 16 == 0 && (p.nk || N % 16 == 0) && width % 8 == 0;
    if (lines) {
        const I8Plan plan = plan_i8(M, N, K, sm_count() > 0 ? sm_count() : 148);
        return plan.pair ? launch_i8_pair(p, plan.tm, plan.split, s) : launch_i8_split(p, plan.tm, plan.split, s);
    }
    return launch_i8_any(p, s);
}

}  // extern "C"
