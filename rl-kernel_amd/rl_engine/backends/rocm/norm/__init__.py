"""Norms between blocks for ROCm gfx950."""
