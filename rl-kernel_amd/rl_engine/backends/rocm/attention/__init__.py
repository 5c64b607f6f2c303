"""Rotary positions and attention over a paged cache for ROCm gfx950."""
