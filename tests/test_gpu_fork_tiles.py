"""Forked requests as test_gpu_fork_step serves them, with the shared prompt read over tiles:
8 heads per KV head are 40 query rows, 24 once two requests have ended, 16 are 80 and 48."""

from __future__ import annotations

import pytest

import test_gpu_fork_step as fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [8, 16])
def test_forked_requests_over_tiles(cuda, monkeypatch, group):
    monkeypatch.setattr(fork, "GROUP", group)
    fork.test_forked_requests_step_by_step(cuda)
