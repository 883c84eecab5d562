from .relative import RelativeAttention
from .sagan import SelfAttention

# registry mirrored from the reference (models/networks/attention/__init__.py:3), plus an attention with heads and positions
ATTENTION_TYPES = {"sagan": SelfAttention, "relative": RelativeAttention}
