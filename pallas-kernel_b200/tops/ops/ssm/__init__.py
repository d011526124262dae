"""Selective state space scan on B200: the recurrence whose decay exp(delta A) and input delta x B
both follow the token, over prompts (``selective_scan``, differentiable) and for single tokens
(``selective_scan_step``)."""
from .scan import selective_scan, selective_scan_step

__all__ = ["selective_scan", "selective_scan_step"]
