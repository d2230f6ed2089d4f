"""Where the norm's outputs may lie: overlaps by which a workgroup would write what another one has yet to read are refused on the host."""
from test_norm_q8_args import norm, q8

AT = 1 << 20        # addresses of buffers that nothing overlaps are multiples of this


def call(d, T=6, **k):
    import bmx
    v = dict(x=AT, residual=None, sum=None, y=3 * AT, rows=None)
    v.update(k)
    return bmx.lib().bmx_rms_norm(d, v["x"], v["residual"], T, v["sum"], v["y"], v["rows"], None), bmx.lib().bmx_last_error()


def refused(d, **k):
    import bmx
    rc, text = call(d, **k)
    assert rc == bmx._lib.BMX_ERR_ARG and b"overlap" in text, (rc, text, k)


def test_outputs_on_inputs():
    row = 64 * 2
    # y on an x of 32 bits: row t of y covers a half of x's row t / 2
    refused(norm(x_dtype=2), y=AT)
    refused(norm(x_dtype=2), y=AT + 6 * 2 * row - 16)
    refused(norm(), y=AT + row)
    refused(norm(), y=AT - row)
    both = dict(residual=5 * AT, sum=7 * AT)
    refused(norm(), **{**both, "y": 5 * AT})
    refused(norm(residual_dtype=0), **{**both, "y": 5 * AT})
    refused(norm(), **{**both, "y": 7 * AT})
    # the sum, of residual's 32 bits, on an x of 16, and beside its rows
    refused(norm(), **{**both, "sum": AT})
    refused(norm(residual_dtype=0), **{**both, "sum": AT + row})
    refused(norm(), **{**both, "sum": 5 * AT + 2 * row})
    # x and its sum in one place leave none there for y
    refused(norm(residual_dtype=0), **{**both, "sum": AT, "y": AT})
    # the weight (at 256)
    refused(norm(), y=256)
    refused(norm(), **{**both, "sum": 256 + 16})


def test_rows_on_anything():
    r = q8(N=6, K=64, codes=9 * AT, scale=11 * AT)
    both = dict(residual=5 * AT, sum=7 * AT, rows=r)
    for place in ("x", "residual", "sum", "y"):
        refused(norm(), **{**both, place: 9 * AT})
        refused(norm(), **{**both, place: 9 * AT + 15 * 64})         # codes lie in blocks of 16 rows
        refused(norm(), **{**both, place: 11 * AT + 16})
    refused(norm(), rows=q8(N=6, K=64, codes=256, scale=11 * AT))
    refused(norm(), rows=q8(N=6, K=64, codes=9 * AT, scale=9 * AT + 64))
