"""Arrays of small elements that the serving kernels read or write as 8- or 16-byte vectors are
declared with that alignment: without it, it is the compiler's choice of place that keeps the
access whole. CPU only."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "proof-carrying-kernels_b200" / "csrc"
VECTOR = {"uint2": 8, "uint4": 16, "float2": 8, "float4": 16}


@pytest.mark.parametrize("name", ["kv4_append.cu", "kv4_attention.cu", "logits_kernel.cu", "lora_kernel.cu"])
def test_arrays_taken_as_vectors_are_aligned(name: str) -> None:
    text = re.sub(r"//.*", "", (CSRC / name).read_text())
    arrays: dict[str, list[int]] = {}
    for line in text.splitlines():
        found = re.match(r"\s*(?:extern )?(?:__shared__ )?(?:(?:alignas|__align__)\((\d+)\) )?"
                         r"(?:const )?(?:T|u?int\d*_t|int|float|uint8_t) (\w+)\[.*\];", line)  # fmt: skip
        if found:
            arrays.setdefault(found[2], []).append(int(found[1] or 1))
    seen = set()
    for kind, array in re.findall(r"reinterpret_cast<(?:const )?(\w+)\*>\((\w+)(?:\[\w+\])?(?: \+ \w+)?\)", text):
        if kind in VECTOR and array in arrays:
            seen.add(array)
            assert min(arrays[array]) >= VECTOR[kind], f"{array} is taken as {kind}"
    assert seen == {"kv4_append.cu": {"e"}, "kv4_attention.cu": {"x"}, "logits_kernel.cu": {"counts"}, "lora_kernel.cu": set()}[name]
