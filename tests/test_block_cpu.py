"""CPU tests of the calls for blocks of 128 and of the rows' ways there and back: what the C ABI refuses before it touches CUDA (made-up
addresses do)."""
import ctypes

A, B, C, D, E, F = (0x1000000 * i for i in range(1, 7))


def test_quantiser_refuses(capi):
    L = capi.load()

    def call(x=A, x_type=0, row_bytes=512, rows=8, k=256, block=0, code_type=0, row_index=None, top_k=0, out_rows=0, codes=B, scales=C):
        return L.catccos_b200_block_quant(None, x, x_type, row_bytes, rows, k, block, code_type, row_index, top_k, out_rows, codes, scales)

    index = dict(row_index=D, top_k=2, out_rows=16)
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(x=A + 8), dict(codes=B + 8), dict(scales=C + 2), dict(k=0), dict(k=24),
                dict(x_type=3), dict(x_type=-1), dict(x_type=2), dict(row_bytes=504), dict(row_bytes=520), dict(row_bytes=1 << 40), dict(rows=2**31),
                dict(block=3), dict(block=-1), dict(code_type=2), dict(code_type=-2), dict(index, block=1), dict(index, block=2), dict(index, top_k=0),
                dict(index, row_index=D + 2), dict(index, out_rows=2**31),
                # overlaps
                dict(codes=A), dict(codes=A + 4080), dict(scales=A + 64), dict(scales=B + 1024), dict(index, codes=D), dict(index, scales=D + 32)):
        assert call(**bad) == -1, bad
    assert call(rows=0, x=None, codes=None) == 0 and call(**dict(index, out_rows=0)) == 0


def _operand(capi, codes, scales, line, transposed=0, per_column=0, type=0, scale_row=1, scale_col=1, matrix=0, scale_matrix=0):
    return capi.BlockOperand(codes=codes, line_bytes=line, matrix_bytes=matrix, scales=scales, scale_row=scale_row, scale_col=scale_col,
                             scale_matrix=scale_matrix, transposed=transposed, per_column=per_column, type=type)


def test_products_refuse(capi):
    L = capi.load()
    m, n, k = 32, 64, 256

    def dense(a=None, b=None, c=E, m=m, n=n, k=k, c_type=0, null=()):
        a = _operand(capi, **{"codes": A, "scales": B, "line": 256, "scale_row": 2, **(a or {})})
        b = _operand(capi, **{"codes": C, "scales": D, "line": 64, **(b or {})})
        return L.catccos_b200_block_gemm(None, None if "a" in null else ctypes.byref(a), None if "b" in null else ctypes.byref(b), c, m, n, k, c_type)

    def grouped(a=None, b=None, offsets=F, c=E, rows=m, experts=3, n=n, k=k, c_type=0):
        a = _operand(capi, **{"codes": A, "scales": B, "line": 256, "scale_row": 2, **(a or {})})
        b = _operand(capi, **{"codes": C, "scales": D, "line": 64, "matrix": 64 * 256, "scale_matrix": 2, **(b or {})})
        return L.catccos_b200_block_grouped_gemm(None, ctypes.byref(a), ctypes.byref(b), offsets, c, rows, experts, n, k, c_type)

    both = [dict(n=0), dict(n=24), dict(k=0), dict(k=24), dict(n=2**31), dict(k=2**31), dict(c=None), dict(c=E + 16), dict(c_type=3), dict(c_type=-2)]
    for operand, codes, scales in (("a", A, B), ("b", C, D)):
        both += [{operand: bad} for bad in (
            dict(codes=None), dict(scales=None), dict(codes=codes + 8), dict(scales=scales + 2), dict(line=48), dict(line=264), dict(line=1 << 40),
            dict(type=2), dict(type=-2), dict(transposed=2), dict(per_column=2), dict(scale_row=1 << 40), dict(scale_col=1 << 40))]
    both += [dict(a=dict(per_column=1)), dict(c=A), dict(c=A + 32 * 256 - 32), dict(c=C + 32), dict(b=dict(scales=E + 64)), dict(a=dict(scales=E + 4092))]
    for bad in both:
        assert dense(**bad) == -1, bad
        assert grouped(**bad) == -1, bad
    for bad in (dict(m=2**31), dict(null="a"), dict(null="b"), dict(a=dict(transposed=1, line=32), m=24), dict(b=dict(per_column=1, scale_row=64, scale_col=2)),
                dict(b=dict(per_column=1, scale_row=66)), dict(b=dict(per_column=1, scale_row=64, scales=D + 8))):
        assert dense(**bad) == -1, bad
    for bad in (dict(experts=0), dict(experts=1025), dict(offsets=None), dict(offsets=F + 2), dict(a=dict(transposed=1, line=32)), dict(b=dict(per_column=1, scale_row=64)),
                dict(b=dict(matrix=0)), dict(b=dict(matrix=64 * 256 - 16)), dict(b=dict(matrix=64 * 256 + 8)), dict(b=dict(scale_matrix=1 << 40)), dict(c=F - 4096 + 32)):
        assert grouped(**bad) == -1, bad
    assert dense(m=0) == 0 and grouped(rows=0) == 0


def test_dispatch_refuses(capi):
    L = capi.load()

    def call(x=A, index=B, out=C, tokens=4, rows=8, n=64, top_k=2):
        return L.catccos_b200_moe_dispatch(None, x, index, out, tokens, rows, n, top_k)

    for bad in (dict(x=None), dict(index=None), dict(out=None), dict(x=A + 8), dict(index=B + 2), dict(out=C + 8), dict(n=0), dict(n=12), dict(top_k=0),
                dict(rows=2**31), dict(out=A), dict(out=B - 16)):
        assert call(**bad) == -1, bad
    assert call(tokens=0) == 0 and call(rows=0) == 0


def test_gradients_refuse(capi):
    L = capi.load()

    def dispatch(d_rows=A, rows=8, index=B, shared=C, out=D, tokens=4, n=64, top_k=2, f16=0):
        return L.catccos_b200_moe_dispatch_grad(None, d_rows, rows, index, shared, out, tokens, n, top_k, f16)

    for bad in (dict(d_rows=None), dict(index=None), dict(out=None), dict(d_rows=A + 8), dict(index=B + 2), dict(shared=C + 8), dict(out=D + 8), dict(n=0),
                dict(n=12), dict(top_k=0), dict(f16=2), dict(f16=-1), dict(rows=2**31), dict(out=A), dict(out=C + 16), dict(out=B - 16)):
        assert dispatch(**bad) == -1, bad
    assert dispatch(tokens=0) == 0

    def combine(d_out=A, y=B, rows=8, index=C, weights=D, d_y=E, d_weights=F, tokens=4, n=64, top_k=2, f16=0):
        return L.catccos_b200_moe_combine_grad(None, d_out, y, rows, index, weights, d_y, d_weights, tokens, n, top_k, f16)

    for bad in (dict(d_out=None), dict(y=None), dict(index=None), dict(weights=None), dict(d_y=None), dict(d_weights=None), dict(d_out=A + 8), dict(y=B + 8),
                dict(index=C + 2), dict(weights=D + 2), dict(d_y=E + 8), dict(d_weights=F + 2), dict(n=0), dict(n=12), dict(top_k=0), dict(f16=2),
                dict(rows=2**31), dict(d_y=A), dict(d_y=B + 16), dict(d_y=C), dict(d_y=D), dict(d_y=F - 16), dict(d_weights=A), dict(d_weights=B + 64),
                dict(d_weights=C + 16), dict(d_weights=D)):
        assert combine(**bad) == -1, bad
    assert combine(tokens=0) == 0
