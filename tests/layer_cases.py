"""Calls of linear and gated_linear that between them run every kernel the products are built for, and which ones a call takes."""
from lmms_engine_amd import _abi

ROWS, STEPS = 0, 1
LAYERS = {"linear": _abi.PRODUCT_LINEAR, "gated": _abi.PRODUCT_GATED}


def product(kind, dtype, m, n, k, a, b, turned=(False, False)):
    """A product of operands given as (strides of a [lines, k] matrix), 16-byte aligned; turned: the reduction runs down the columns."""
    p = _abi.Product(kind=kind, dtype=dtype, m=m, n=n, k=k)
    for f, strides, turn in (("a", a, turned[0]), ("b", b, turned[1])):
        row, col = strides[::-1] if turn else strides
        getattr(p, f)[:] = (1 << 20, 1 << 20)
        getattr(p, f + "_row")[:] = (row, row)
        getattr(p, f + "_col")[:] = (col, col)
    p.out[:] = (1 << 20, 1 << 20)
    return p


def lay(rows, cols, transposed):
    return (1, rows) if transposed else (cols, 1)


def products(layer, dtype, t, k, n, x_transposed, w_transposed):
    """{pass: product} of a call and of its backward pass."""
    x, w, dz = lay(t, k, x_transposed), lay(n, k, w_transposed), (-(-n // 8) * 8, 1)
    gated = layer == "gated"
    return {"forward": product(LAYERS[layer], dtype, t, n, k, x, w),
            "dx": product(_abi.PRODUCT_SUM if gated else _abi.PRODUCT_LINEAR, dtype, t, k, n, dz, w, (False, True)),
            "dw": product(_abi.PRODUCT_EACH if gated else _abi.PRODUCT_LINEAR, dtype, n, k, t, dz, x, (True, True))}


def kernel(p, cus=256):
    """(dtype, tile, threads, order of the left operand, of the right one, gated) and whether the reduction is split."""
    r = _abi.product_route(p, cus)
    order = {_abi.OPERAND_ROWS: ROWS, _abi.OPERAND_STEPS: STEPS, _abi.OPERAND_ROWS_COPIED: ROWS, _abi.OPERAND_STEPS_COPIED: STEPS, _abi.OPERAND_GATHERED: ROWS}
    return (p.dtype, r.tile, r.threads, order[r.a], order[r.b], p.kind == _abi.PRODUCT_GATED), r.parts > 1


# dtype code, tokens, inner, outer: every kernel of every pass with four k-tiles at least, whole reductions and split ones, ragged and whole sizes
EVERY_KERNEL = [(_abi.F32, 72, 4100, 4100), (_abi.F32, 136, 136, 136), (_abi.F32, 136, 2819, 4100), (_abi.F32, 2819, 72, 2056), (_abi.F32, 2819, 72, 4100),
                (_abi.F32, 2819, 136, 4100), (_abi.F32, 2819, 4100, 136), (_abi.BF16, 72, 1500, 72), (_abi.BF16, 72, 6150, 1500),
                (_abi.BF16, 136, 4100, 6150), (_abi.BF16, 203, 1032, 6150), (_abi.BF16, 203, 2819, 4100), (_abi.BF16, 264, 517, 4100),
                (_abi.BF16, 1001, 203, 4100), (_abi.BF16, 1500, 72, 72), (_abi.BF16, 2819, 203, 4100), (_abi.BF16, 2819, 2819, 203),
                (_abi.BF16, 4100, 136, 2819), (_abi.BF16, 4100, 136, 6150), (_abi.BF16, 6150, 329, 329), (_abi.BF16, 6150, 1032, 203),
                # a result of many whole and ragged 256-tiles over 16 k-tiles, and sizes of blocks in use
                (_abi.BF16, 4099, 1000, 4100), (_abi.BF16, 512, 1024, 2816), (_abi.BF16, 600, 896, 4864)]
