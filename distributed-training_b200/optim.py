"""Reference module name ``dtrain.optim``."""
from .ops.optim import AdamW, clip_grads, clip_scale, global_norm  # noqa: F401
