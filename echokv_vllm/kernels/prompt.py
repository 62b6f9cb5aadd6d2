"""``echokv_vllm.kernels.prompt``: the module ``echokv_amd.kernels.prompt`` beside the reference's names."""

import sys

from echokv_amd.kernels import prompt as _module

sys.modules[__name__] = _module
