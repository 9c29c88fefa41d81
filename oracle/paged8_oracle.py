# SPDX-License-Identifier: Apache-2.0
"""8-bit paged KV-cache oracle: the format and its storing in 64 bits on the CPU, run by run."""
from __future__ import annotations

import math

import torch

LARGEST = {"e4m3": 448.0, "int8": 127.0}
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def round_code(x: torch.Tensor, held: str) -> torch.Tensor:
    """float64 values over their scale to the nearest code, ties to even."""
    if held == "int8":
        return x.round()
    ex = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.pow(2.0, ex - 3)
    return (x / step).round() * step


def exponent(top: float, held: str) -> float:
    """Of the smallest scale for magnitudes up to `top`; NaN where there is none."""
    if not math.isfinite(top):
        return math.nan
    for e in range(-60, 61):
        if held == "e4m3" and top <= 448 * 2.0 ** e:
            return e
        if held == "int8" and round(top / 2.0 ** e) <= 127:
            return e
    return math.nan


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """What codes [pages, H, page, D] with exponents [pages, H, page / block] stand for, float64."""
    block = codes.shape[2] // exps.shape[2]
    return codes.double() * torch.pow(2.0, exps).repeat_interleave(block, 2)[..., None]


def exps_of(scales: torch.Tensor) -> torch.Tensor:
    raw = scales.cpu().view(torch.uint8).double()
    return torch.where(raw == 255, math.nan, raw - 127)


def bytes_of(exps: torch.Tensor) -> torch.Tensor:
    return torch.where(torch.isnan(exps), 255.0, exps + 127).to(torch.uint8)


def store(codes: torch.Tensor, exps: torch.Tensor, new: torch.Tensor, slots, held: str) -> None:
    """Rows [N, H, S, D] to slots, in place: codes float64 [pages, H, page, D], exps float64 [pages, H, page / block]."""
    pages, H, page, D = codes.shape
    block = page // exps.shape[2]
    rows = new.double().transpose(1, 2).reshape(-1, H, D)
    runs = []  # (first slot, its tokens)
    for t, s in enumerate(slots):
        if not 0 <= s < pages * page:
            continue
        if runs and t > 0 and slots[t - 1] == s - 1 and s % block:
            runs[-1][1].append(t)
        else:
            runs.append((s, [t]))
    for s, tokens in runs:
        at, inside = s // page, s % page
        first = inside % block
        for h in range(H):
            x = rows[tokens, h]
            e = exponent(float("nan") if torch.isnan(x).any() else x.abs().max().item(), held)
            if first:
                was = exps[at, h, inside // block].item()
                e = math.nan if math.isnan(e) or math.isnan(was) else max(e, was)
                kept = slice(inside - first, inside)
                if math.isnan(e):
                    codes[at, h, kept] = 0
                elif e > was:
                    codes[at, h, kept] = round_code(codes[at, h, kept] * 2.0 ** (was - e), held)
            exps[at, h, inside // block] = e
            codes[at, h, inside: inside + len(tokens)] = 0 if math.isnan(e) else round_code(x * 2.0 ** -e, held)
