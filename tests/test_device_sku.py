"""The SKU that a gfx950 part's peak engine clock names, where the clock reads a little off (no GPU here)."""
from __future__ import annotations

import sys
from types import SimpleNamespace

import pytest

from teamredbench_amd import device


@pytest.mark.parametrize("clock, sku", [(2400, "MI355X"), (2402, "MI355X"), (2403, "MI355X"), (2390, "MI355X"),
                                        (2205, "MI350X"), (2300, None), (2500, None), ("N/A", None)])
def test_sku_by_peak_engine_clock(monkeypatch, clock, sku):
    smi = SimpleNamespace(
        AmdSmiClkType=SimpleNamespace(GFX="gfx"), amdsmi_init=lambda: None, amdsmi_shut_down=lambda: None,
        amdsmi_get_processor_handles=lambda: ["h"], amdsmi_get_gpu_device_bdf=lambda h: "0000:0a:00.0",
        amdsmi_get_gpu_board_info=lambda h: {"product_name": "N/A"},
        amdsmi_get_gpu_asic_info=lambda h: {"market_name": "AMD Radeon Graphics"},
        amdsmi_get_clock_info=lambda h, kind: {"max_clk": clock})
    monkeypatch.setitem(sys.modules, "amdsmi", smi)
    props = SimpleNamespace(pci_domain_id=0, pci_bus_id=0x0A, pci_device_id=0, gcnArchName="gfx950:sramecc+:xnack-")
    torch_like = SimpleNamespace(cuda=SimpleNamespace(get_device_properties=lambda i: props))
    names = device._amdsmi_names(torch_like, 0)
    assert names[0] == "AMD Radeon Graphics" and len(names) == (1 if sku is None else 2)
    assert sku is None or sku in names[1]
