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


def test_windows_of_wide_tables():
    """A sequence's ranges are no more than the workgroups that run at once over kv
    heads and turns of rows, whatever the tables' width."""
    lib = _lib.load()

    def size(total_q, max_q, hq, hk, width, keys=0, block=256):
        return lib.mskv_window_weights_bounded_workspace_bytes(total_q, max_q, keys, hq, hk,
                                                               block, width)
    row = 32 * 4
    # 64 windows of 64 queries under tables of a million tokens: 256 rows a kv head
    assert size(64 * 64, 64, 32, 8, 4096) == 64 * 64 * row * (32 + 1) + 4
    assert size(32, 32, 32, 8, 4096) == 32 * row * (64 + 1) + 4
    assert size(32, 32, 32, 8, 4096, keys=1000) == 32 * row * (4 + 1) + 4
    assert size(5, 5, 32, 32, 1) == 5 * row * 2 + 4
    # a step of a decode that reads K again: a query a sequence
    splits = lib.mskv_decode_num_splits(256, 32, 8, 4096, 256)
    assert (lib.mskv_decode_weights_workspace_bytes(256, 32, 8, 256, 4096)
            == lib.mskv_decode_workspace_bytes(256, 32, 8, 128, splits))
    # the bound of any heads holds every call's
    whole = lib.mskv_window_weights_workspace_bytes
    assert whole(4096, 0, 32, 256, 4096) == 4096 * row * (512 + 1) + 4
    for hk in (1, 2, 8, 32):
        for max_q in (1, 64, 4096):
            for width in (1, 7, 500, 4096):
                assert size(4096, max_q, 32, hk, width) <= whole(4096, 0, 32, 256, width)
    assert size(0, 0, 32, 8, 4) == size(4, 4, 30, 8, 4) == size(4, -1, 32, 8, 4) == 0
