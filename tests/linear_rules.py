"""The rules by which csrc/linear.hip chooses a kernel, for operands that start on 16-byte boundaries: tests name with them which
kernel a size is meant to reach, so that a change of a rule cannot silently leave a kernel untested."""


def _up(a, b):
    return -(-a // b)


def _choose(rows16, acol, M, N, splits, size, cus):
    tn = _up(N, 128) * splits
    if _up(M, 128) * tn < cus // 2:
        return "tile64"
    if size == 4 and not acol and max(_up(M, 64) * _up(N, 64), cus) * 29 < max(_up(M, 128) * tn, cus) * 67:
        return "tile64"
    if not rows16:
        return "tile128"
    large = 256 if acol else 192
    few_large = _up(_up(M, large) * tn, cus) * large * 100 <= _up(_up(M, 128) * tn, cus) * 128 * 115
    return f"stream{large if few_large else 128}"


def _rows16(size, *lds):
    return all(ld * size % 16 == 0 and ld < 1 << 20 for ld in lds)


def forward(rows, K, N, size, cus):
    if rows <= 4:
        return "few"
    tile = _choose(_rows16(size, K, N), False, rows, N, 1, size, cus)
    if tile == "tile64":
        def cost(r, t):
            n = _up(rows, r) * _up(N, r)
            return (_up(n, cus) * cus if r == 32 else max(n, cus)) * t
        c64, c32, c16 = cost(64, 41 if size == 2 else 72), cost(32, 21), cost(16, 10)
        two = c32 * 11 < c64 * 10
        if c16 * 11 < (c32 if two else c64) * 10:
            return "shared16"
        if two:
            return "shared32"
    return tile


def splits(rows, K, N, size, cus):
    large = size == 2 or _rows16(size, N, K)
    tiles = _up(N, 256 if large else 128) * _up(K, 128)
    want = cus // tiles
    if want * tiles * 16 < cus * 15 or rows > 1280 * want:
        want = 2 * cus // tiles
    want = max(1, min(want, rows // 256))
    span = max(64, _up(_up(rows, want), 64) * 64)
    return _up(rows, span)


def backward(rows, K, N, size, cus):
    """-> the kernels of dx = dz W and of dW = dz^T x, the latter with its splits of the rows."""
    n = splits(rows, K, N, size, cus)
    dx = _choose(_rows16(size, N, K), False, rows, K, 1, size, cus)
    dw = _choose(_rows16(size, N, K), True, N, K, n, size, cus)
    return dx, dw + (" split" if n > 1 else "")
