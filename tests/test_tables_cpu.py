"""The module that fills AdamW's host tables: a missing one, one of another build and a buffer of another size are refused."""
import ctypes as C
import sys
import types

import pytest
import torch

import psgd_pro_amd as P
from psgd_pro_amd import _lib as L

NAME = "psgd_pro_amd._tables"


@pytest.fixture
def fresh(monkeypatch):
    monkeypatch.setattr(L, "_tables", None)
    return monkeypatch


def call():
    x = torch.zeros(3)
    P.adamw_step([x], [x], [x], [x], step=1)


def test_the_built_module_is_the_bindings_own(fresh):
    assert L.tables().VERSION == L.TABLES_VERSION and L.tables() is L.tables()


def test_a_missing_module_says_how_to_build_it(fresh):
    fresh.setitem(sys.modules, NAME, None)
    with pytest.raises(RuntimeError, match="build it with"):
        call()


@pytest.mark.parametrize("version", [None, L.TABLES_VERSION - 1, L.TABLES_VERSION + 1])
def test_a_module_of_another_build_fills_nothing(fresh, version):
    def adamw(*args):
        raise AssertionError("called")

    stale = types.SimpleNamespace(adamw=adamw, changed=adamw, __file__="_tables.so")
    if version is not None:
        stale.VERSION = version
    fresh.setitem(sys.modules, NAME, stale)
    with pytest.raises(RuntimeError, match="rebuild it with"):
        call()


@pytest.mark.parametrize("count", [0, 7, 9, 16, -8])
def test_a_buffer_of_another_size_is_refused(count):
    x, buf = torch.zeros(3), (C.c_int64 * 16)()
    with pytest.raises(RuntimeError, match="numbers expected"):
        L.tables().adamw([x], [x], [x], [x], C.addressof(buf), count)
    assert not any(buf)
