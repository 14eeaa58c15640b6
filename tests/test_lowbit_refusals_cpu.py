"""What the low-bit C entries refuse before anything is launched (no GPU here)."""


def test_expand_refuses_views_that_share_rows():
    from taomate_hd_amd import _native

    lib, ok = _native.load(), 4096  # stands for an aligned address that is never read
    views = (_native.KV8Segment * 3)()
    for i, n in enumerate((100, 64, 65)):
        views[i] = _native.KV8Segment(4096, 4096, 4096, 4096, 128, 0, n, i % 2)

    def expand(*dst):
        return lib.tmhd_kv8_expand(views, (_native.c_int32 * 3)(*dst), 3, ok, ok, 512 * 64, 512 * 64, 512, 2, 64, None)

    # blocks taken: two, one, two; (0, 128, 192) shares none
    for dst in ((0, 0, 192), (0, 64, 192), (64, 0, 64), (128, 192, 256), (0, 128, 128), (256, 0, 192)):
        assert expand(*dst) == _native.TMHD_ERR_INVALID and b"share rows" in lib.tmhd_last_error(), dst
    # a place outside of the slot, behind views that share none: the other refusal
    assert expand(0, 128, 512) == _native.TMHD_ERR_INVALID and b"share rows" not in lib.tmhd_last_error()
