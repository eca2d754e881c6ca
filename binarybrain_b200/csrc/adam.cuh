// One parameter's step of Adam (cuda/OptimizerAdam.cu:12-48), as the plain and the clipped optimizer kernels take it.
#pragma once

namespace bb200 {

__device__ __forceinline__ void adam_step(float &p, float g, float &m, float &v, float lr_t, float beta1, float beta2)
{
    m += (1.0f - beta1) * (g - m);
    v += (1.0f - beta2) * (g * g - v);
    p -= lr_t * m / (sqrtf(v) + 1.0e-7f);
}

}   // namespace bb200
