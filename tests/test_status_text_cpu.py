"""The text of the error that a device status turns into: every bit has its words, and none is left out."""
import re
from pathlib import Path

import pytest

from qwen3_triton import _abi

HEADER = Path(__file__).resolve().parent.parent / 'include' / 'q3b200.h'
BITS = {name: int(bit) for name, bit in re.findall(r'Q3_(STATUS_\w+) = (\d+)', HEADER.read_text())}


def text_of(monkeypatch, value):
    monkeypatch.setattr(_abi, 'read_status', lambda device=None: value)
    with pytest.raises(_abi.Q3Error) as error:
        _abi.raise_on_status()
    return str(error.value)


def test_every_bit_of_the_header_has_words(monkeypatch):
    assert len(BITS) == 6 and all(getattr(_abi, name) == bit for name, bit in BITS.items())
    texts = [text_of(monkeypatch, bit) for bit in BITS.values()]
    assert all(re.fullmatch(r'device status: \S.{5,}', text) for text in texts) and len(set(texts)) == len(texts)
    assert 'capacity' in text_of(monkeypatch, _abi.STATUS_CACHE_RANGE)
    assert 'not held' in text_of(monkeypatch, _abi.STATUS_CACHE_RECENT)


def test_several_bits_and_unknown_ones(monkeypatch):
    both = text_of(monkeypatch, _abi.STATUS_ID_RANGE | _abi.STATUS_CACHE_RECENT)
    assert 'embedding id' in both and 'not held' in both
    assert '0x400' in text_of(monkeypatch, 0x400) and 'label' in text_of(monkeypatch, 0x402)
    monkeypatch.setattr(_abi, 'read_status', lambda device=None: 0)
    _abi.raise_on_status()
