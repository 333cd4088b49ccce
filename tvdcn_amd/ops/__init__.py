"""tvdcn_amd.ops -- the names of tvdcn.ops (tvdcn/ops/__init__.py), and operators on channels-last maps."""
from .activations import *  # noqa: F401,F403
from .deform_conv import *  # noqa: F401,F403
from .deform_conv_transpose import *  # noqa: F401,F403
from .dropout import *  # noqa: F401,F403
from .group_norm import *  # noqa: F401,F403
from .int8_maps import *  # noqa: F401,F403
from .pointwise import *  # noqa: F401,F403
from .pointwise_int8 import *  # noqa: F401,F403
from .rms_norm import *  # noqa: F401,F403
