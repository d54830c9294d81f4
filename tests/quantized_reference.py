"""The microscaled formats by their definition, in 64 bits and on the CPU: what
``iekv.engine.quantized`` holds of a row, and what its bytes stand for."""
from __future__ import annotations

import torch

GROUP, LEAST = 32, -100
LARGEST = {"mxfp8": 448.0, "mxint8": 127.0, "mxfp4": 6.0}
FORMATS = list(LARGEST)


def _e4m3(code: int) -> float:
    field, part = code >> 3 & 15, code & 7
    size = (1 + part / 8) * 2.0 ** (field - 7) if field else part / 8 * 2.0 ** -6
    return float("nan") if code & 127 == 127 else -size if code & 128 else size


# The value of every code; of e2m1 codes 0..15.
CODES = {"mxfp8": torch.tensor([_e4m3(c) for c in range(256)], dtype=torch.float64),
         "mxint8": torch.tensor([c - 256 if c > 127 else c for c in range(256)],
                                dtype=torch.float64),
         "mxfp4": torch.tensor([s * m for s in (1, -1) for m in (0, .5, 1, 1.5, 2, 3, 4, 6)],
                               dtype=torch.float64)}


def _power(e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones((), dtype=torch.float64), e)


def _rounded(y: torch.Tensor, format: str) -> torch.Tensor:
    """The code of the value nearest to each y; of two the one whose last bit is 0."""
    values = CODES[format]
    codes = torch.arange(len(values))
    usable = torch.isfinite(values) & (values.abs() <= LARGEST[format])
    # The positive ones in order, even codes among equals of a distance.
    codes = codes[usable & (values >= 0) & ~((values == 0) & (codes > 0))]
    values = values[codes]
    size = y.abs()
    above = torch.searchsorted(values, size).clamp(max=len(values) - 1)
    below = (above - 1).clamp(min=0)
    near, far = values[above] - size, size - values[below]
    take = torch.where(near == far, codes[above] % 2 == 0, near < far)
    code = torch.where(take, codes[above], codes[below])
    if format == "mxint8":
        return torch.where(y < 0, (256 - code) % 256, code)
    return code + torch.signbit(y) * (8 if format == "mxfp4" else 128)


def encode(rows: torch.Tensor, format: str) -> torch.Tensor:
    """[..., D] values as records, uint8."""
    x = rows.detach().cpu().double()
    dim = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -dim % GROUP)).unflatten(-1, (-1, GROUP))
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, 0.0)
    most = x.abs().amax(-1)
    # From one or two below what the logarithm says: the smallest that suffices.
    e = torch.log2(most / LARGEST[format]).floor().clamp(min=LEAST + 1).long() - 1
    for _ in range(3):
        e = torch.where(most > LARGEST[format] * _power(e), e + 1, e)
    y = x / _power(e)[..., None]
    codes = _rounded(y.flatten(-2)[..., :dim].contiguous(), format)
    codes = torch.where(finite.repeat_interleave(GROUP, -1)[..., :dim], codes, 0)
    if format == "mxfp4":
        codes = codes[..., 0::2] + 16 * codes[..., 1::2]
    scales = torch.where(finite, e + 127, 255)
    scales = torch.nn.functional.pad(scales, (0, 4 - scales.shape[-1]))
    return torch.cat((codes, scales), -1).to(torch.uint8)


def decode(records: torch.Tensor, format: str) -> torch.Tensor:
    """Records as the values they stand for, [..., D] in float64."""
    records = records.cpu().long()
    codes, scales = records[..., :-4], records[..., -4:]
    if format == "mxfp4":
        codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    scale = torch.where(scales == 255, float("nan"), _power(scales - 127)).repeat_interleave(GROUP, -1)
    return CODES[format][codes] * scale[..., :codes.shape[-1]]


def same_records(got: torch.Tensor, want: torch.Tensor, format: str) -> bool:
    """Equal bytes, the sign of a zero apart."""
    got, want = got.cpu(), want.cpu()
    return torch.equal(got[..., -4:], want[..., -4:]) and torch.equal(
        code_values(got, format), code_values(want, format))


def code_values(records: torch.Tensor, format: str) -> torch.Tensor:
    codes = records[..., :-4].long()
    if format == "mxfp4":
        codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    return CODES[format][codes]
