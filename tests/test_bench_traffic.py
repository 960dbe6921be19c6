"""The committed counter profile and the kernel sources it belongs to, on the CPU."""

from __future__ import annotations

import os

import bench

CSRC = os.path.join("mini-llm-runtime_amd", "csrc")


def test_the_committed_profile_is_of_these_sources():
    traffic, source = bench.measured_traffic()
    assert traffic is not None, source
    assert traffic["decode_step_bytes"] > 0 and traffic["prefill_call_bytes"] > 0
    assert os.path.exists(os.path.join(bench.REPO, source))


def test_sources_of_other_kernels_do_not_make_a_profile_stale(tmp_path, monkeypatch):
    (tmp_path / CSRC).mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / CSRC / "paged_decode.hip").write_text("decode")
    monkeypatch.setattr(bench, "REPO", str(tmp_path))
    sha = bench.kernel_sources_hash()
    for name in bench.UNPROFILED_SOURCES:
        (tmp_path / CSRC / name).write_text("another kernel")
    assert bench.kernel_sources_hash() == sha
    (tmp_path / CSRC / "paged_decode.h").write_text("its header")
    assert bench.kernel_sources_hash() != sha


def test_those_sources_exist_and_hold_no_profiled_kernel():
    csrc = os.path.join(bench.REPO, CSRC)
    others = [n for n in os.listdir(csrc) if n not in bench.UNPROFILED_SOURCES]
    for name in bench.UNPROFILED_SOURCES:
        assert os.path.exists(os.path.join(csrc, name))
    for name in others:
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        assert not any(f'"{header}"' in text for header in bench.UNPROFILED_SOURCES), name
