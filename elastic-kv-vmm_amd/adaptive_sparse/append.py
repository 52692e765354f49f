"""New tokens into the paged pool (HIP): keys and queries rotated by their positions, K/V rows and 8-bit index keys written.

The reference leaves the rotation and the K/V store to its engine and only
records what was stored (adaptive_sparse/logical_shadow.py:44-70). Here one
launch of csrc/append.hip rotates a layer's queries and keys and writes K and V
through the slot map that extend_block_tables made, with its positions; a
second operator writes the index keys that select_blocks scores blocks with.
"""

import math
from dataclasses import dataclass, field
from fractions import Fraction

import torch

from elastic_kv import _native

from .kv_pool import KVPlanes
from .profile_ranges import profile_range

SCALINGS = (None, "linear", "base", "ramp")


@dataclass(frozen=True)
class Rotary:
    """How a head's first 2 * len(turns) elements turn with the position (make_rotary)."""

    turns: torch.Tensor      # int64: turns a position of every pair, times 2^64, modulo 2^64
    magnitude: float         # factor of the rotated elements
    interleaved: bool        # pairs are elements 2i and 2i + 1 instead of i and i + len(turns)
    frequencies: tuple = field(repr=False)   # radians a position


def _power(base, exponent):
    try:
        return base ** exponent
    except OverflowError:
        return math.inf


def _held(frequencies):
    if not all(math.isfinite(f) for f in frequencies):
        raise ValueError("frequencies must be finite")
    return frequencies


def rotary_frequencies(rotary_dim, *, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """(radians a position of every pair, factor of the rotated elements) of make_rotary's arguments."""
    if type(rotary_dim) is not int or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    base, factor = float(base), float(factor)
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError("base and factor must be positive")
    if scaling == "base":
        if rotary_dim < 4:
            raise ValueError("scaling the base needs a rotary_dim of 4 or more")
        base *= _power(factor, rotary_dim / (rotary_dim - 2))
        if not 0 < base < math.inf:
            raise ValueError("the scaled base must be positive and finite")
    plain = _held([_power(base, -2 * i / rotary_dim) for i in range(rotary_dim // 2)])
    if scaling == "linear":
        return _held([f / factor for f in plain]), 1.0
    if scaling != "ramp":
        return plain, 1.0
    if original is None or not (math.inf > original > 0 and math.inf > fast > slow > 0 and base > 1):
        raise ValueError("a ramp needs the original context length, fast > slow > 0 and a base above 1")
    # The place among the pairs of one that turns `turns` times in the original context.
    place = [rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
    low, high = max(math.floor(place[0]), 0), min(math.ceil(place[1]), rotary_dim - 1)
    slowed = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rotary_dim // 2)]
    return _held([f * (1 - s) + f / factor * s for f, s in zip(plain, slowed)]), max(0.1 * math.log(factor) + 1.0, 1.0)


def make_rotary(rotary_dim, *, device, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0,
                magnitude=None, interleaved=False):
    """A Rotary of `rotary_dim` elements: pair i of rotary_dim / 2 turns by base ** (-2i / rotary_dim) radians a position.

    scaling, for contexts longer than those a model was trained on: "linear"
    divides the frequencies by `factor`; "base" raises the base by
    factor ** (rotary_dim / (rotary_dim - 2)), which divides the slowest one;
    "ramp" keeps the pairs that turn more than `fast` times in the `original`
    context, divides those that turn less than `slow` times, and goes linearly
    from one to the other between them, with a magnitude of 0.1 ln(factor) + 1
    (Peng et al., "YaRN: Efficient context window extension of large language
    models", 2023). magnitude: another factor of the rotated elements.

    A frequency and its turns are rounded as numbers of 64 bits: where a pair
    turns a radian a position or less, its angle is off by less than 4e-16
    radians a position, 4e-7 at position 2^30.
    """
    frequencies, factor_of = rotary_frequencies(rotary_dim, base=base, scaling=scaling, factor=factor,
                                                original=original, fast=fast, slow=slow)
    turns = []
    for f in frequencies:
        whole = round(Fraction(f / (2 * math.pi)) * 2 ** 64) % 2 ** 64
        turns.append(whole - 2 ** 64 if whole >= 2 ** 63 else whole)
    return Rotary(torch.tensor(turns, dtype=torch.int64, device=device),
                  float(factor_of if magnitude is None else magnitude), bool(interleaved), tuple(frequencies))


@profile_range("native/append_rotary")
def append_rotary(query, key, value, planes, slots, positions, rotary, output, *, page_size=1, layer=0, zero_below=1):
    """Rotate queries into `output` and keys into the pool by `positions`; write K and V rows to `slots`.

    query, output [N, Hq, D], key, value [N, Hkv, D] bfloat16 or float16, dense
    in D (slices of one projection, for instance); output may be the query.
    positions, slots [N] int32 or int64, as extend_block_tables writes them; a
    token with position < 0 is left out, and a slot below zero_below or past
    the pool writes no row. Slots of live tokens are distinct. rotary: a Rotary
    of at most D elements (make_rotary); the others are copied. planes: the
    pool's KVPlanes, a plane row holding a token ([Hkv, D]) or a whole page
    ([page_size, Hkv, D]). query and output may be None (keys and values only),
    or key, value, planes and slots (rotation only).
    """
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary (make_rotary)")
    if planes is not None and not isinstance(planes, KVPlanes):
        raise TypeError("planes must be a KVPlanes")
    helper, entries = _native.launch_helper()
    status = helper.append_rotary(entries["ekv_append_rotary"], query, key, value, planes, layer, page_size, slots,
                                  zero_below, positions, rotary.turns, rotary.magnitude, rotary.interleaved, output)
    _native.launch_check(status, "append_rotary")


@profile_range("native/append_index")
def append_index(index_key, planes, scales, slots, *, page_size=1, layer=0, zero_below=1):
    """Write index keys as 8-bit whole numbers to `slots`, and each row's scale to scales[slot].

    index_key [N, Di] bfloat16 or float16, finite (rotated already, if it is
    to be: append_rotary); planes: KVPlanes of one plane a layer (kv 1) whose
    rows hold a token's Di bytes, or a whole page's; scales: float32, one for
    each slot of the layer. A row's scale is its largest magnitude / 127, its
    codes are the quotients by it, rounded to whole numbers (halves to even).
    Slots below zero_below or past the pool write nothing.
    """
    if not isinstance(planes, KVPlanes):
        raise TypeError("planes must be a KVPlanes")
    helper, entries = _native.launch_helper()
    status = helper.append_index(entries["ekv_append_index"], index_key, planes, layer, page_size, scales, slots,
                                 zero_below)
    _native.launch_check(status, "append_index")
