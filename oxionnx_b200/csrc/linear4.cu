// Rows times a matrix of 4-bit codes with a scale (and a zero point) for each group of inputs: a warp for each output of
// each row, sums in f32.
#include "decoder_device.cuh"

namespace oxb {
namespace k {

namespace {

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) linear4_outputs(Linear4 a) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t out = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (out >= a.rows * a.n) return;
  const int64_t m = out / a.n, j = out % a.n;
  float sum = 0.f;
  for (int g = 0; g < a.groups; ++g) {
    const int64_t at = j * a.groups + g;
    const uint8_t zb = a.zeros ? a.zeros[j * ((a.groups + 1) / 2) + g / 2] : 0;
    const float zero = a.zeros ? (float)(g & 1 ? zb >> 4 : zb & 15) : 8.f;
    float part = 0.f;
    for (int i = lane; i < a.group; i += 32) {
      const int kk = g * a.group + i;
      if (kk >= a.k) break;
      const uint8_t c = a.codes[at * (a.group / 2) + i / 2];
      part += to_f32(((const T*)a.x)[m * a.k + kk]) * ((float)(i & 1 ? c >> 4 : c & 15) - zero);
    }
    sum += part * a.scales[at];
  }
  for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) ((T*)a.y)[out] = from_f32<T>(a.bias ? sum + a.bias[j] : sum);
}

}  // namespace

void linear4(const Linear4& a, cudaStream_t s) {
  if (a.rows == 0) return;
  const dim3 grid((unsigned)ceil_div(a.rows * a.n, kWarps));
  if (a.dt == DT::F32) launch(linear4_outputs<float>, grid, dim3(kWarps * 32), 0, s, a);
  else if (a.dt == DT::F16) launch(linear4_outputs<__half>, grid, dim3(kWarps * 32), 0, s, a);
  else launch(linear4_outputs<__nv_bfloat16>, grid, dim3(kWarps * 32), 0, s, a);
}

}  // namespace k
}  // namespace oxb
