"""The widest row of scores that draws take, refused on the host before any launch (no GPU needed)."""
import ctypes as C


def test_sample_codes_takes_at_most_two_to_the_nineteen_codes():
    import __graft_entry__ as g
    g.build()
    from mqgan_amd import _lib
    lib, at = _lib.load(), C.c_void_p(4096)
    for codes in ((1 << 19) + 1, 1 << 20):
        d = _lib.SampleDesc(rows=1, row_stride=codes, codes=codes, dtype=0, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
        assert lib.mq_sample_codes(C.byref(d), at, at, None, None, None, None, None, at, None, None) != 0
        assert b"at most 2^19" in lib.mq_last_error()
