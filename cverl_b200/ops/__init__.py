"""Hot ops: hand-written sm_100a kernels behind autograd functions, each with a PyTorch oracle."""
from .gemm import gemm_nn, gemm_nt, gemm_tn_acc, linear, launch_counter  # noqa: F401
from .norm import add_rmsnorm, gated_rmsnorm, headnorm_rope, rmsnorm, rope_tables  # noqa: F401
from .activation import conv1d_silu, conv1d_silu_split, embedding, siggate, swiglu  # noqa: F401
from .lmhead import lmhead_logprob  # noqa: F401
from .fp8 import (Fp8Tensor, Fp8Weight, add_rmsnorm_fp8, add_rmsnorm_linear_fp8, gemm_fp8_nt,  # noqa: F401
                  linear_fp8, quantize_fp8, quantize_fp8_pair, quantize_fp8_t, quantize_fp8_weight)
from . import rl, optim  # noqa: F401
