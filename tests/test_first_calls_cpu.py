"""Threads whose first calls of the 4-bit products or the rotary positions meet: the
second one either finds the tables of types whole or makes them itself."""
from __future__ import annotations

import threading

import pytest


class Torch:
    """torch, with `meanwhile` run in another thread at the n-th attribute taken."""

    def __init__(self, torch, n, meanwhile):
        self.torch, self.left, self.meanwhile = torch, n, meanwhile

    def __getattr__(self, name):
        self.left -= 1
        if self.left == 0:
            thread = threading.Thread(target=self.meanwhile)
            thread.start()
            thread.join()
        return getattr(self.torch, name)


def refusals(torch, llk, name):
    """A call that the last of its checks refuses, with operands on the CPU."""
    if name == "q4":
        codes = torch.zeros(32, 4, dtype=torch.uint8)
        with pytest.raises(ValueError, match="scales"):
            llk.Q4Weights.from_codes(codes, torch.zeros(1, 4))
    else:
        table = llk.RotaryTable(8, device="cpu")
        table.device_index = 5
        x = torch.zeros(2, 1, 8)
        with pytest.raises(ValueError, match="table"):
            llk.rotary(x, None, torch.zeros(2, dtype=torch.int32), table)


@pytest.mark.parametrize("nth", range(1, 10))
@pytest.mark.parametrize("name,tables", [("q4", ("_BF16", "_BYTES", "_SCALES", "_SUMS", "_OUT")),
                                         ("positions", ("_FLOATS", "_INT32"))])
def test_first_calls_of_two_threads(llk, monkeypatch, name, tables, nth):
    import importlib

    import torch
    module = importlib.import_module(f"dslcompiler_amd.{name}")
    for table in tables:
        monkeypatch.setattr(module, table, None)
    monkeypatch.setattr(module, "_begin", lambda: -1)  # the device of a CPU tensor
    errors = []

    def meanwhile():
        monkeypatch.setattr(module, "_torch", lambda: torch)
        try:
            refusals(torch, llk, name)
        except BaseException as e:  # noqa: BLE001 (pytest's own failure among them)
            errors.append(e)

    monkeypatch.setattr(module, "_torch", lambda: Torch(torch, nth, meanwhile))
    refusals(torch, llk, name)
    assert not errors
