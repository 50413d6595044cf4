"""How far a gfx950 part's reported peak engine clock may lie from the one that names its SKU (no GPU here)."""
from __future__ import annotations

import sys
from types import SimpleNamespace

import pytest

from teamredbench_amd import device


def _names(monkeypatch, clock) -> list[str]:
    smi = SimpleNamespace(
        AmdSmiClkType=SimpleNamespace(GFX="gfx"), amdsmi_init=lambda: None, amdsmi_shut_down=lambda: None,
        amdsmi_get_processor_handles=lambda: ["h"], amdsmi_get_gpu_device_bdf=lambda h: "0000:0a:00.0",
        amdsmi_get_gpu_board_info=lambda h: {"product_name": "N/A"},
        amdsmi_get_gpu_asic_info=lambda h: {"market_name": "AMD Radeon Graphics"},
        amdsmi_get_clock_info=lambda h, kind: {"max_clk": clock})
    monkeypatch.setitem(sys.modules, "amdsmi", smi)
    props = SimpleNamespace(pci_domain_id=0, pci_bus_id=0x0A, pci_device_id=0, gcnArchName="gfx950:sramecc+:xnack-")
    torch_like = SimpleNamespace(cuda=SimpleNamespace(get_device_properties=lambda i: props))
    return device._amdsmi_names(torch_like, 0)[1:]


@pytest.mark.parametrize("clock", [2380, 2389, 2406, 2420, 2180, 2189, 2206, 2220])
def test_a_clock_that_was_never_read_names_no_sku(monkeypatch, clock):
    """A clock of the moment on its way down must not make an MI355X an MI350X."""
    assert _names(monkeypatch, clock) == []


@pytest.mark.parametrize("clock, sku", [(2400, "MI355X"), (2402, "MI355X"), (2403, "MI355X"), (2200, "MI350X")])
def test_the_name_holds_the_clock_that_was_read(monkeypatch, clock, sku):
    (name,) = _names(monkeypatch, clock)
    assert sku in name and f"read as {clock}" in name
