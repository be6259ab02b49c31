// The MX4 quantisation's kernel and the C interface of the MX4 tensors as host code, around the stand-ins of tests/simt_emu.cu: a
// launch of the quantisation runs its blocks as host threads, a product is only written down.  The tests look at what each
// call lets the launch behind it do, which no run on a GPU shows reliably.
//
// Built as a shared library by tests/test_mx4_order_of_launches.py.
#include <type_traits>

#include "simt_emu.cu"

#include <cmath>
#include <string>

namespace emu {

std::atomic<unsigned int> released{0};    // calls that let the launch behind start

inline uint32_t shfl_xor_bits(uint32_t value, unsigned int mask)
{
    shift = mask;
    return exchange(value, [](unsigned int lane) { return lane ^ shift; });
}

inline uint32_t vmaxu2(uint32_t a, uint32_t b)
{
    return std::max(a & 0xFFFFu, b & 0xFFFFu) | std::max(a >> 16, b >> 16) << 16;
}

// nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code
inline uint32_t e2m1(float v)
{
    const float middle[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.0f};
    uint32_t code = 0;
    for (uint32_t i = 0; i < 7; ++i) {
        code += (i + 1) % 2 == 0 ? std::fabs(v) >= middle[i] : std::fabs(v) > middle[i];
    }
    return code | (std::signbit(v) ? 8u : 0u);
}

inline uint32_t e2m1x8(const float (&v)[8])
{
    uint32_t word = 0;
    for (uint32_t i = 0; i < 8; ++i) {
        word |= e2m1(v[i]) << (4 * i);
    }
    return word;
}

inline float half_value(uint32_t code)
{
    const float values[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    return (code & 8u) != 0u ? -values[code & 7u] : values[code & 7u];
}

inline uint32_t half_pair(uint32_t byte)
{
    const __half2 pair = __floats2half2_rn(half_value(byte & 15u), half_value(byte >> 4));
    uint32_t bits;
    std::memcpy(&bits, &pair, 4);
    return bits;
}

inline void f16x2_e2m1(uint32_t codes, uint32_t (&out)[4])
{
    for (uint32_t i = 0; i < 4; ++i) {
        out[i] = half_pair(codes >> (8 * i) & 255u);
    }
}

inline void f16x2_e2m1_4(unsigned short codes, uint32_t &low, uint32_t &high)
{
    low = half_pair(codes & 255u);
    high = half_pair(codes >> 8);
}

} // namespace emu

#undef __shfl_xor_sync
#define __shfl_xor_sync(mask, value, lanes) emu::shfl_xor_bits((value), (lanes))
#define __vmaxu2(a, b) emu::vmaxu2((a), (b))
#define __float_as_uint(v) emu::float_as_uint(v)
#define grid_launch_dependents() ((void)++emu::released)

namespace emu {
inline uint32_t float_as_uint(float value)
{
    uint32_t bits;
    std::memcpy(&bits, &value, 4);
    return bits;
}
} // namespace emu

#include "mx4_ptx.cuh"
#define cvt_e2m1x8(v) emu::e2m1x8(v)
#define cvt_f16x2_e2m1(codes, out) emu::f16x2_e2m1((codes), (out))
#define cvt_f16x2_e2m1_4(codes, low, high) emu::f16x2_e2m1_4((codes), (low), (high))
#include "mx4_quant.cu"

// ---- the launches that do not run here ------------------------------------------------------------
namespace q8 {
static std::string product;    // the last product's description, whole

cudaError_t launch_mx4_product(cudaStream_t, const UmmaScratch &, unsigned int, unsigned int, const Mx4Product &p)
{
    product.assign(reinterpret_cast<const char *>(&p), sizeof(p));
    return cudaSuccess;
}

bool mx4_linear_quantizes(uint32_t, uint32_t, uint32_t m, unsigned int)
{
    return m <= 4u;
}

cudaError_t launch_mx4_order(cudaStream_t, bool, const uint32_t *, uint32_t, const uint32_t *, uint32_t, uint32_t, uint32_t *,
                             uint32_t *, uint32_t *)
{
    return cudaSuccess;
}
} // namespace q8

// (the device of the calling thread is device 0, as far as the interface can see)
#define cudaGetDevice(device) (*(device) = 0, cudaSuccess)
#define cudaSetDevice(device) ((void)(device), cudaSuccess)
#include "mx4_api.cu"

extern "C" void *mx4_emu_context()
{
    aotx_q8_ctx *ctx = new aotx_q8_ctx();
    ctx->sm_count = 148;
    ctx->overlap = 1;
    return ctx;
}

extern "C" void mx4_emu_release(void *ctx)
{
    delete static_cast<aotx_q8_ctx *>(ctx);
}

extern "C" unsigned int mx4_emu_released()
{
    return emu::released.exchange(0u);
}

extern "C" size_t mx4_emu_product(char *to, size_t room)
{
    const size_t bytes = q8::product.size() < room ? q8::product.size() : room;
    std::memcpy(to, q8::product.data(), bytes);
    q8::product.clear();
    return bytes;
}
