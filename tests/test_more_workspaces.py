"""The workspaces of shared prefixes and windows follow what their launches can use."""

from microserve_amd import _lib


def _shared(batch, hq, prefix=8192, hk=8, block=256, width=64, groups=1):
    return _lib.load().mskv_shared_decode_workspace_bytes(batch, groups, hq, hk, block, width,
                                                          prefix)


def test_shared_prefixes_of_large_batches():
    """The ranges of a prefix that run at once are fewer the more rows read it."""
    partial = 129 * 4
    assert _shared(64, 32) <= 64 * 32 * (64 + 32) * partial + 64 * 4 + 256
    for batch, hq in ((256, 32), (512, 32), (512, 64), (1024, 32)):
        assert _shared(batch, hq) < 300 << 20, (batch, hq)
        assert _shared(batch, hq, prefix=1 << 30) < 300 << 20, (batch, hq)
    # past that a few partials a row, as the decode's splits
    for batch in (2048, 8192, 65535):
        assert _shared(batch, 32) <= batch * 32 * 12 * partial + batch * 4 + 256, batch
