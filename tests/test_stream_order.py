"""Work that a launch depends on is enqueued on the launch's own stream (CPU only, on the sources).

A handle's stream is non-blocking, so nothing orders it behind the null stream: memory cleared there (hipMemset,
which may return before it has written) can still be cleared after a kernel on the handle's stream has counted in it."""
import os
import re

import pytest

from mvlm_amd import build


def text(path):
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def test_the_handles_stream_is_not_ordered_behind_the_null_stream():
    assert "hipStreamNonBlocking" in text(os.path.join(build.CSRC, "runtime.cpp"))


@pytest.mark.parametrize("path", build.sources(), ids=os.path.basename)
def test_device_memory_is_cleared_on_the_handles_stream(path):
    t = text(path)
    assert not re.search(r"\bhipMemset(D8|D16|D32)?\s*\(", t)
    for call in re.findall(r"\bhipMemset\w*Async\s*\(([^;]*?)\)\s*(?:[;,]|!=|==)", t):
        assert call.rstrip(" )").endswith("dev->stream"), call
