"""``echokv_vllm.kernels.shared``: the module ``echokv_amd.kernels.shared`` beside the reference's names."""

import sys

from echokv_amd.kernels import shared as _module

sys.modules[__name__] = _module
