// snk_optim.hpp — AdamW handle internals shared by snk_optim.hip and snk_dqn.hip / snk_trainer.hip
#pragma once
#include "snk_common.hpp"

namespace snk {
snk_adamw adamw_create(int32_t n, const int64_t *sizes, const float *wd, const snk_adamw_cfg_t *cfg);
void adamw_not_captured(hipStream_t s, const char *what);   // throws where s is being captured
void adamw_free(snk_adamw h);
void adamw_bind(snk_adamw h, void *const *params, const void *const *grads, void *const *copies, hipStream_t s);
// grads: this step's own, of type grad_dtype; nullptr: as bound
void adamw_step(snk_adamw h, float lr, float grad_scale, hipStream_t s, int32_t grad_dtype = SNK_F32,
                const void *const *grads = nullptr);
void adamw_reset(snk_adamw h, hipStream_t s);   // zero moments, step 0
void adamw_set_owned(snk_adamw h);              // a model's: destroy and bind refuse it
}  // namespace snk
