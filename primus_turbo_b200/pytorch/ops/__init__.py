from .gemm_fp8 import *  # noqa: F401,F403
from .grouped_gemm_fp8 import *  # noqa: F401,F403
from .int4 import *  # noqa: F401,F403
from .quantization import *  # noqa: F401,F403
