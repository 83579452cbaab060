"""Per-shape constant tables of the forward, built once per (grid, text length) on the host
and kept on the device, as the reference engine does (src/iris_metal/model.py:147-174).

- rotary tables: FP32 ``cos``/``sin`` ``[N, 64]`` for the trunk in ``[text | image]`` order and
  ``[L, 64]`` for the pixel stage (src/iris3b/nn/rope.py:19-89);
- the pixel stage's fixed 2-D sincos position table, stored separably as ``[W, 8]`` (x half)
  and ``[H, 8]`` (y half) since each half depends on one coordinate
  (src/iris3b/nn/embeddings.py:269-288);
- the frequencies of ``kernels.rotary``, plain or scaled for long contexts;
- the timestep frequency bank ``exp(-ln(P) k / n)`` (src/iris3b/nn/embeddings.py:41-45).
"""

from __future__ import annotations

import math

import torch


def rope_2d_angles(head_dim: int, height: int, width: int, theta: float, scale: float, aspect: str,
                   frame_pairs: int = 0, frame_theta: float = 10.0, frame_index: int = 0) -> torch.Tensor:
    """Complex ``[H*W, head_dim/2]`` table of src/iris3b/nn/rope.py:19-82 (x, y pairs interleaved)."""
    n_pairs = head_dim // 4
    if not 0 <= frame_pairs < n_pairs:
        raise ValueError(f"rope: frame_pairs={frame_pairs} is not one of 0..{n_pairs - 1}")
    freqs = 1.0 / theta ** (torch.arange(0, head_dim, 4)[:n_pairs].float() / head_dim)
    freqs = freqs[: n_pairs - frame_pairs]
    if aspect == "square":
        xs, ys = torch.linspace(0, scale, width), torch.linspace(0, scale, height)
    elif aspect == "isotropic":
        step = scale / max(max(height, width) - 1, 1)
        xs, ys = torch.arange(width).float() * step, torch.arange(height).float() * step
    else:
        raise ValueError(f"rope: aspect must be 'square' or 'isotropic', got {aspect!r}")
    x_cis = torch.polar(torch.ones(width, freqs.numel()), torch.outer(xs, freqs))
    y_cis = torch.polar(torch.ones(height, freqs.numel()), torch.outer(ys, freqs))
    cis = torch.stack(
        [x_cis[None, :, :].expand(height, width, -1), y_cis[:, None, :].expand(height, width, -1)], dim=-1
    ).reshape(height * width, -1)
    if frame_pairs:
        slots = 2 * frame_pairs
        f_freqs = 1.0 / frame_theta ** (torch.arange(slots).float() / slots)
        f_cis = torch.polar(torch.ones(slots), float(frame_index) * f_freqs)
        cis = torch.cat([cis, f_cis[None, :].expand(height * width, -1)], dim=-1)
    return cis


def rope_1d_angles(head_dim: int, length: int, theta: float) -> torch.Tensor:
    """Complex ``[length, head_dim/2]`` table of src/iris3b/nn/rope.py:85-89."""
    freqs = 1.0 / theta ** (torch.arange(0, head_dim, 2)[: head_dim // 2].float() / head_dim)
    ang = torch.outer(torch.arange(length).float(), freqs)
    return torch.polar(torch.ones_like(ang), ang)


def rotary_frequencies(dim: int, theta: float, device, scaling: str = "none", scale: float = 1.0,
                       trained: int = 4096, slow: float = 1.0, fast: float = 32.0) -> tuple[torch.Tensor, float]:
    """``(freqs, factor)`` of ``kernels.rotary``: FP64 ``[dim / 2]`` angles per position of the pairs of a
    ``dim``-wide rotated part, ``theta ** (-2 i / dim)``, and the factor on the rotated values.

    For contexts ``scale`` times the ``trained`` positions: ``"linear"`` divides every angle by ``scale``;
    ``"ntk"`` raises the base so that the slowest pair is divided by ``scale`` and the fastest stays;
    ``"by_parts"`` keeps pairs that turn at least ``fast`` times over the trained positions, divides those
    that turn at most ``slow`` times by ``scale``, blends linearly in the number of turns between them, and
    sets the factor to ``0.1 ln(scale) + 1`` (it meets itself in q k: the scores' temperature)."""
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_frequencies: the rotated width must be even and positive, got {dim}")
    if scaling not in ("none", "linear", "ntk", "by_parts"):
        raise ValueError(f"rotary_frequencies: scaling must be none, linear, ntk or by_parts, got {scaling!r}")
    if scale < 1.0 or (scaling == "none" and scale != 1.0) or not theta > 1.0 or not fast > slow:
        raise ValueError("rotary_frequencies: needs scale >= 1 (1 without scaling), theta > 1 and fast > slow")
    i = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    freqs, factor = theta ** -i, 1.0
    if scaling == "linear":
        freqs = freqs / scale
    elif scaling == "ntk" and dim > 2:
        freqs = (theta * scale ** (dim / (dim - 2))) ** -i
    elif scaling == "by_parts":
        turns = trained * freqs / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freqs = freqs * keep + freqs / scale * (1 - keep)
        factor = 0.1 * math.log(scale) + 1.0
    return freqs.to(device), factor


def cos_sin(*tables: torch.Tensor, device) -> tuple[torch.Tensor, torch.Tensor]:
    cis = torch.view_as_real(torch.cat(tables))
    return cis[..., 0].contiguous().to(device), cis[..., 1].contiguous().to(device)


def sincos_halves(dim: int, height: int, width: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    """``([W, dim/2], [H, dim/2])`` FP32: ``[sin | cos]`` of the column / row coordinate,
    computed in FP64 then rounded, as src/iris3b/nn/embeddings.py:269-288."""
    half = dim // 2
    omega = torch.arange(half // 2, dtype=torch.float64) / (half / 2.0)
    omega = 1.0 / 10000.0**omega

    def one(n: int) -> torch.Tensor:
        out = torch.outer(torch.arange(n, dtype=torch.float32).double(), omega)
        return torch.cat([torch.sin(out), torch.cos(out)], dim=1).float().contiguous()

    return one(width).to(device), one(height).to(device)


def timestep_freqs(freq_dim: int, max_period: float, device) -> torch.Tensor:
    n = freq_dim // 2
    k = torch.arange(n, dtype=torch.float32)
    return torch.exp(-math.log(max_period) * k / n).to(device)
