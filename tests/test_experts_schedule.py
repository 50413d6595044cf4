"""The grouped products' load order and waits, replayed on the host (CPU).

A wave's loads complete in issue order, and a wait for vmcnt <= n leaves the n
newest in flight. The replay issues the prologue and the steps as the kernels
do, for every ring they are built with, and checks at every step that what the
step reads has landed, and that nothing is loaded into a slot that has yet to
be read."""
from __future__ import annotations

from pathlib import Path
import shutil
import subprocess

import pytest

TESTS = Path(__file__).resolve().parent
STEPS = 60


@pytest.fixture(scope="module")
def rings(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    exe = tmp_path_factory.mktemp("schedule") / "experts_schedule_host"
    subprocess.run([hipcc, "--offload-host-only", "-O1", "-std=c++20", "-w", str(TESTS / "experts_schedule_host.cpp"),
                    "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    return [tuple(int(v) for v in line.split()) for line in out.splitlines()]


def _replay(px, nx, ix, py, ny, iy, odd, even, prologue) -> str | None:
    """What goes wrong, or None."""
    operands = [("x", px, nx, ix), ("y", py, ny, iy)]
    issued: list[tuple[str, int]] = []   # (operand, pair or stage) of every load, in order

    def issue(step):
        for name, pairs, slots, loads in operands:
            if pairs and step % 2 == 0:
                continue
            index = (step - 1) // 2 + slots if pairs else step + slots
            if index >= 0:
                issued.extend([(name, index)] * loads)
                old = index - slots   # what the slot held: read during step last - 1, so free from step `last` on
                if old >= 0 and step < (2 * old + 1 if pairs else old):
                    return f"step {step}: {name} {index} overwrites {old} before it is read"
        return None

    for v in range(-2 * max(nx, ny), 0):
        if (wrong := issue(v)) is not None:
            return wrong

    def landed(stage, left):
        done = issued[:len(issued) - left] if left else issued
        for name, pairs, _, loads in operands:
            index = stage // 2 if pairs else stage
            if done.count((name, index)) != loads:
                return f"stage {stage}: {name} {index} has not landed"
        return None

    if (wrong := landed(0, prologue)) is not None:
        return wrong
    for step in range(STEPS):
        if (wrong := landed(step + 1, odd if step % 2 else even)) is not None:   # what the step reads
            return wrong
        if (wrong := issue(step)) is not None:
            return wrong
    return None


def test_every_ring(rings):
    assert len(rings) == 9
    for ring in rings:
        assert _replay(*ring) is None, ring


def test_a_laxer_wait_is_caught(rings):
    for ring in rings:
        *head, odd, even, prologue = ring
        assert _replay(*head, odd + 1, even, prologue) or _replay(*head, odd, even + 1, prologue), ring
        assert _replay(*head, odd, even, prologue + 1), ring
