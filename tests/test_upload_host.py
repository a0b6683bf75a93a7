"""The convenience copies of Cuda, without a device: that their copies have ended when they
return."""
import numpy as np
import pytest

import llmpager_amd as lp


class Recorder(lp.Cuda):
    def __init__(self):
        self.did, self.under_way = [], {}

    def __del__(self):
        pass

    def alloc_device(self, nbytes):
        self.did.append(("alloc", nbytes))
        return 4096

    def htod_async(self, dst, src, stream=None):
        assert src.flags.c_contiguous
        self.under_way[stream] = dst
        self.did.append(("copy", dst, src.nbytes))

    def sync_stream(self, s=None):
        self.under_way.pop(s, None)


@pytest.mark.parametrize("stream", [None, 77])
@pytest.mark.parametrize("a", [np.arange(12, dtype=np.float32), np.arange(24).reshape(4, 6)[:, ::2], np.zeros(0, np.int32)])
def test_uploads_have_ended(a, stream):
    """A stream of the caller's does not wait for the null stream's copy, and the copy may be
    of an array that ends with the call."""
    c = Recorder()
    assert c.upload(a, stream) == 4096
    assert c.did == [("alloc", max(a.nbytes, 1)), ("copy", 4096, a.nbytes)]
    assert not c.under_way
