"""MI355X-native vector quantizer: drop-in for the reference's vqvae.ema_vector_quantizer."""
from .ema_vector_quantizer import EMAVectorQuantizer, LazyOneHot  # noqa: F401
from .boundary import QuantizerBoundary  # noqa: F401
from .projection import Linear, linear  # noqa: F401
from .gradients import clip_grad_norm_, clip_grads, grad_norm  # noqa: F401

__all__ = ["EMAVectorQuantizer", "LazyOneHot", "QuantizerBoundary", "Linear", "linear", "grad_norm", "clip_grads",
           "clip_grad_norm_"]
__version__ = "0.1.0"
