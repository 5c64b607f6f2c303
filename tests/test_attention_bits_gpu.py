"""The stored output bits of paged attention (tests/golden/attention_bits.json, written by tests/golden/make_attention_bits.py on an
MI355X): a build whose kernels add in another order under the same contract id fails here."""

from __future__ import annotations

import importlib.util
import json
from pathlib import Path

import pytest

GOLDEN = Path(__file__).parent / "golden"


@pytest.mark.gpu
def test_attention_reproduces_the_stored_bits_of_its_contract_id():
    spec = importlib.util.spec_from_file_location("make_attention_bits", GOLDEN / "make_attention_bits.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.attention_bits() == json.loads((GOLDEN / "attention_bits.json").read_text())


def test_the_stored_id_is_the_librarys(rlk_lib):
    assert list(json.loads((GOLDEN / "attention_bits.json").read_text())) == [rlk_lib.rlk_attention_contract_id().decode()]
