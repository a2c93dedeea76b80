"""trigrad_amd -- MI355X (gfx950) implementation of trigrad's differentiable tile
rasterizer behind the reference's Python entry point (`render`, `precision`)."""
from . import camera
from .tests_wrapper import barycentric, interpolate3_scalar, interpolate3_vector
from ._C import force_tickets, set_precision, verify_frames
from .adamw import AdamW, adamw_step
from .attention import linear_attention, linear_attention_step
from .norm import group_norm
from .recurrence import linear_recurrence, linear_recurrence_step
from .wrapper import Renderer, precision, render

__all__ = ["render", "barycentric", "interpolate3_scalar", "interpolate3_vector", "precision", "Renderer", "camera", "set_precision",
           "verify_frames", "force_tickets", "linear_recurrence", "linear_recurrence_step", "group_norm",
           "linear_attention", "linear_attention_step", "adamw_step", "AdamW"]

__version__ = "0.1.0"
