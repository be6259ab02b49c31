"""MX4 tensors and the products over them (include/aotx_mx4_b200.h), as methods of `Q8Context`.

An MX4 tensor is rows of k values in blocks of 32 that share a scale, a power of two; a value is one of 0, 0.5, 1, 1.5, 2, 3,
4, 6 with a sign, times the scale of its block: 4.25 bits a value, multiplied by the tensor cores as they are.  Weights are
laid out once with `mx4_quantize` (of a model file's rows: `dequant` gives them as binary16); activations with the
same call or, `mx4_linear`, on their way into a product.

Every method enqueues on the current CUDA stream of PyTorch for the context's device and returns without synchronising.  Like
the rest of the context's methods they are for one thread at a time; tensors used on several streams are ordered by the caller.
A product may read its weights while the operation ahead of it on the stream is still running: what writes them just before it is
`mx4_quantize`, or launches do not overlap (`set_overlap`).
"""
EPILOGUE_STORE, EPILOGUE_ADD, EPILOGUE_SWIGLU = EPILOGUES = 0, 1, 2
# The library's limits.  (It takes 32-bit numbers, and what is larger would be cut on the way: it is refused before.)
MAX_DEPTH, MAX_ROWS, MAX_EXPERTS = 1 << 24, (1 << 31) - 1, 256


_module = None
_words = ()


def _torch():
    global _module, _words
    if _module is None:
        import torch
        _words = (torch.int32, torch.uint32)
        _module = torch
    return _module


class Mx4Tensor:
    """`rows` rows of k values: codes uint8 [rows][k / 2] (value 2i in the low four bits of byte i), scales uint8
    [ceil(k / 128)][rows][4] (byte b of (c, r): values 128c + 32b .. of row r, 2^(byte - 127); 255 is NaN; 0 past k).

    It shares the storage of the two tensors that it is made of, as a view does: what is written there later is read, storage
    that grows under it is followed."""
    __slots__ = ("rows", "k", "device", "_codes", "_scales", "_bytes", "_behind")

    def __init__(self, codes, scales):
        torch = _torch()
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError("codes and scales are uint8, codes [rows][k / 2]")
        self.rows, self.k = codes.shape[0], 2 * codes.shape[1]
        if self.k == 0 or self.k % 32 != 0 or tuple(scales.shape) != ((self.k + 127) // 128, self.rows, 4):
            raise ValueError("k is a multiple of 32 and scales are [ceil(k / 128)][rows][4]")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device:
            raise ValueError("codes and scales lie without gaps on one device")
        if self.k > MAX_DEPTH or self.rows > MAX_ROWS:
            raise ValueError("%d rows of %d values" % (self.rows, self.k))
        self.device = codes.device
        # (views of its own: neither another storage for the caller's tensors (`.data = ...`) nor another shape changes what it reads)
        self._codes, self._scales = codes.detach(), scales.detach()
        self._bytes = None

    @classmethod
    def empty(cls, rows, k, device):
        """Both arrays in one allocation."""
        if k <= 0 or k % 32 != 0 or rows < 0:
            raise ValueError("k is a multiple of 32")
        t = cls._make(rows, k, device)
        t.device = t._bytes.device
        return t

    @classmethod
    def _make(cls, rows, k, device):
        if k > MAX_DEPTH or rows > MAX_ROWS:
            raise ValueError("%d rows of %d values" % (rows, k))
        torch = _torch()
        t = cls.__new__(cls)
        t.rows, t.k = rows, k
        # (a row of codes is a multiple of 16 bytes, so the scales behind them lie on such a boundary too)
        t._behind = codes = rows * (k // 2)
        t._bytes = torch.empty(codes + (k + 127) // 128 * rows * 4, dtype=torch.uint8, device=device)
        t.device = device
        return t

    @property
    def codes(self):
        if self._bytes is None:
            return self._codes.detach()
        return self._bytes[:self._behind].view(self.rows, self.k // 2)

    @property
    def scales(self):
        if self._bytes is None:
            return self._scales.detach()
        return self._bytes[self._behind:].view((self.k + 127) // 128, self.rows, 4)

    def _addresses(self):
        """Where codes and scales are now: `resize_` of a tensor with the same storage may have put it elsewhere."""
        held = self._bytes
        if held is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = held.data_ptr()
        return at, at + self._behind


def _pointer(t):
    return t.data_ptr() if t is not None else None


_codes = {}


def _dtype_code(dtype):
    code = _codes.get(dtype)
    if code is None:
        torch = _torch()
        _codes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        code = _codes.get(dtype)
        if code is None:
            raise ValueError("float32, float16 or bfloat16, not %s" % dtype)
    return code


class Mx4Calls:
    """The part of Q8Context that works on MX4 tensors."""

    def _mx4_linear_bytes_call(self, *args):
        return self.lib.aotx_mx4_linear_workspace_bytes(*args)

    def _mx4_elsewhere(self, t):
        return ValueError("a tensor on %s, a context for %s" % (t.device, self.device))

    def _mx4_words(self, what, t, count=None):
        """The address of a device array of 32-bit whole numbers, or none."""
        if t is None:
            return None
        if t.dtype not in _words or not t.is_contiguous():
            raise ValueError("%s is int32 or uint32 without gaps" % what)
        if count is not None and t.numel() != count:
            raise ValueError("%s has %d entries, not %d" % (what, t.numel(), count))
        if t.device != self.device:
            raise self._mx4_elsewhere(t)
        return t.data_ptr()

    def _mx4_rows_in(self, x):
        """Rows of 16- or 32-bit values: their number, their length, the distance of rows."""
        shape = x.shape
        if len(shape) != 2 or shape[1] == 0 or shape[1] % 32 != 0:
            raise ValueError("x is [rows][k], k a multiple of 32")
        rows, k = shape
        if x.device != self.device:
            raise self._mx4_elsewhere(x)
        if x.is_contiguous():
            return rows, k, k
        apart, side = x.stride()
        if side != 1 or (rows > 1 and apart < k):
            raise ValueError("the values of a row lie side by side and rows do not overlap")
        return rows, k, max(apart, k)

    def _mx4_result(self, y, rows, n, y_dtype, epilogue):
        """y of `rows` rows for n rows of weights, the caller's or a new one, and the code of its type."""
        if epilogue not in EPILOGUES:
            raise ValueError("unknown epilogue")
        width = self._mx4_width(n, epilogue) if epilogue == EPILOGUE_SWIGLU else n
        if y is None:
            if epilogue == EPILOGUE_ADD:
                raise ValueError("EPILOGUE_ADD adds into a y that the caller gives")
            torch = _module or _torch()
            if y_dtype is None:
                y_dtype = torch.float32
            code = _codes.get(y_dtype)
            if code is None:
                code = _dtype_code(y_dtype)
            return torch.empty(rows, width, dtype=y_dtype, device=self.device), code
        if y.shape != (rows, width) or not y.is_contiguous() or (y_dtype is not None and y.dtype != y_dtype):
            raise ValueError("y is [%d][%d] without gaps" % (rows, width))
        if y.device != self.device:
            raise self._mx4_elsewhere(y)
        return y, _dtype_code(y.dtype)

    def _mx4_width(self, n, epilogue):
        if epilogue == EPILOGUE_SWIGLU:
            if n % 2 != 0:
                raise ValueError("gate and up rows come in pairs")
            return n // 2
        return n

    def _mx4_pair(self, w, k, x=None):
        if w.k != k:
            raise ValueError("rows of %d and of %d values" % (w.k, k))
        # (one object for one device, so that the next call need not compare them)
        if w.device is not self.device:
            if w.device != self.device:
                raise self._mx4_elsewhere(w)
            w.device = self.device
        if x is not None and x.device is not self.device:
            if x.device != self.device:
                raise self._mx4_elsewhere(x)
            x.device = self.device

    # -- quantisation -----------------------------------------------------------------------------------------------
    def mx4_quantize(self, x, rows=None, rows_dev=None, out=None):
        """Rows of x (float32, float16, bfloat16; rows may lie apart) as an Mx4Tensor.  `rows`: int32 row numbers of x, one
        for each row of the result (a number outside x leaves its row as it was).  `rows_dev`: device word with the
        live number of rows."""
        code = _codes.get(x.dtype)
        if code is None:
            code = _dtype_code(x.dtype)
        have, k, stride = self._mx4_rows_in(x)
        count = have if rows is None else rows.numel()
        if out is None:
            out = Mx4Tensor._make(count, k, self.device)
        elif out.rows != count or out.k != k:
            raise ValueError("out has %d rows of %d values" % (out.rows, out.k))
        elif out.device != self.device:
            raise self._mx4_elsewhere(out)
        codes, scales = out._addresses()
        result = self._mx4_quantize_call(
            self._address, self._stream(), x.data_ptr(), code, have, stride, k,
            None if rows is None else self._mx4_words("rows", rows), count,
            None if rows_dev is None else self._mx4_words("rows_dev", rows_dev, 1), codes, scales)
        if result != 0:
            self._check(result)
        return out

    def mx4_dequant(self, t, first_row=0, rows=None, out=None, dtype=None):
        """The values of rows first_row .. first_row + rows of an MX4 tensor, float16 unless `dtype` or `out` says otherwise."""
        torch = _torch()
        rows = t.rows - first_row if rows is None else rows
        if first_row < 0 or rows < 0 or first_row + rows > t.rows:
            raise ValueError("rows %d .. %d of %d" % (first_row, first_row + rows, t.rows))
        if t.device != self.device:
            raise self._mx4_elsewhere(t)
        if out is None:
            dtype = dtype or torch.float16
            code = _dtype_code(dtype)
            out = torch.empty(rows, t.k, dtype=dtype, device=self.device)
        else:
            code = _dtype_code(out.dtype)
            if tuple(out.shape) != (rows, t.k) or not out.is_contiguous() or (dtype is not None and out.dtype != dtype):
                raise ValueError("out is [%d][%d] without gaps" % (rows, t.k))
            if out.device != self.device:
                raise self._mx4_elsewhere(out)
        codes, scales = t._addresses()
        result = self._mx4_dequant_call(self._address, self._stream(), codes, scales, t.rows, t.k, first_row, rows,
                                        out.data_ptr(), code)
        if result != 0:
            self._check(result)
        return out

    # -- products ---------------------------------------------------------------------------------------------------
    def mx4_matmul(self, w, x, m_dev=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE):
        """y[m][n] = x . w^T for two MX4 tensors; `m_dev`, `y` and `epilogue` as in `matmul_fused`."""
        self._mx4_pair(w, x.k, x)
        y, y_code = self._mx4_result(y, x.rows, w.rows, y_dtype, epilogue)
        w_codes, w_scales = w._addresses()
        x_codes, x_scales = x._addresses()
        result = self._mx4_matmul_call(self._address, self._stream(), w_codes, w_scales, w.rows, w.k, x_codes, x_scales, x.rows,
                                       None if m_dev is None else self._mx4_words("m_dev", m_dev, 1), y.data_ptr(),
                                       y_code, epilogue)
        if result != 0:
            self._check(result)
        return y

    def mx4_linear(self, w, x, m_dev=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE, workspace=None):
        """`mx4_matmul` of w with `mx4_quantize(x)`, up to the order of the float sums; few rows are quantised by the kernel
        that multiplies them."""
        code = _codes.get(x.dtype)
        if code is None:
            code = _dtype_code(x.dtype)
        m, k, stride = self._mx4_rows_in(x)
        self._mx4_pair(w, k)
        y, y_code = self._mx4_result(y, m, w.rows, y_dtype, epilogue)
        if workspace is None:
            size = self._mx4_linear_bytes_call(self._address, w.rows, k, m)
            if size:
                torch = _torch()
                workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        else:
            size = workspace.numel() * workspace.element_size()
            if not workspace.is_contiguous():
                raise ValueError("the workspace has gaps")
            if workspace.device != self.device:
                raise self._mx4_elsewhere(workspace)
        w_codes, w_scales = w._addresses()
        result = self._mx4_linear_call(self._address, self._stream(), w_codes, w_scales, w.rows, k, x.data_ptr(), code, stride,
                                       m, None if m_dev is None else self._mx4_words("m_dev", m_dev, 1), y.data_ptr(),
                                       y_code, epilogue, _pointer(workspace), size)
        if result != 0:
            self._check(result)
        return y

    # -- routed experts ---------------------------------------------------------------------------------------------
    def moe_order(self, ids, experts, tokens_dev=None):
        """The (token, rank) pairs of ids [tokens][used] by expert: order (the pair at each place), their tokens, and
        offsets [experts + 1] of the experts' places; int32, places that no pair has hold -1."""
        torch = _torch()
        shape = ids.shape
        if len(shape) != 2 or shape[1] == 0:
            raise ValueError("ids is [tokens][used]")
        tokens, used = shape
        pairs = tokens * used
        if experts <= 0 or experts > MAX_EXPERTS or pairs > MAX_ROWS:
            raise ValueError("%d selections of %d experts" % (pairs, experts))
        at = self._mx4_words("ids", ids)
        # (one allocation and one split: slices of it take 0.7 us more, three allocations 0.3)
        words = torch.empty(2 * pairs + experts + 1, dtype=torch.int32, device=self.device)
        order, token_of, offsets = words.split_with_sizes((pairs, pairs, experts + 1))
        base = words.data_ptr()
        result = self._mx4_order_call(self._address, self._stream(), at, tokens, self._mx4_words("tokens_dev", tokens_dev, 1),
                                      used, experts, base, base + 4 * pairs, base + 8 * pairs)
        if result != 0:
            self._check(result)
        return order, token_of, offsets

    def mx4_matmul_grouped(self, w, experts, x, offsets, y_rows=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE):
        """Rows offsets[e] .. offsets[e + 1] of x times expert e's rows of w (w.rows / experts each).  `y_rows`: int32, the row
        of y for each row of x (one outside y is left out).  Rows that no expert has are not written."""
        self._mx4_pair(w, x.k, x)
        if experts <= 0 or experts > MAX_EXPERTS or w.rows % experts != 0:
            raise ValueError("%d rows of w for %d experts" % (w.rows, experts))
        if epilogue == EPILOGUE_ADD:
            raise ValueError("grouped products store or apply the gated unit")
        n = w.rows // experts
        if y is not None and y.dim() != 2:
            raise ValueError("y is [rows][%d]" % self._mx4_width(n, epilogue))
        rows = x.rows if y is None or y_rows is None else y.shape[0]
        if rows >= 1 << 32:
            raise ValueError("%d rows of y" % rows)
        y, y_code = self._mx4_result(y, rows, n, y_dtype, epilogue)
        w_codes, w_scales = w._addresses()
        x_codes, x_scales = x._addresses()
        result = self._mx4_grouped_call(self._address, self._stream(), w_codes, w_scales, experts, n, w.k, x_codes, x_scales,
                                        x.rows, self._mx4_words("offsets", offsets, experts + 1),
                                        self._mx4_words("y_rows", y_rows, x.rows), rows, y.data_ptr(), y_code,
                                        epilogue)
        if result != 0:
            self._check(result)
        return y

    def mx4_moe_ffn(self, w_gate_up, w_down, experts, x, prob, ids, tokens_dev=None, out=None, out_dtype=None):
        """The routed feed-forward step of `moe_ffn_fused` on MX4 weights (gate and up rows of an expert interleaved): the
        pairs in the experts' order, their rows of x quantised, gate and up by expert with the gated unit, its
        result (in x's type, which has to hold it: binary16 up to 65504) quantised, the down product by expert, and the
        rank-ordered weighted sum.  x is any type that `mx4_quantize` takes; prob [tokens][experts] float32 and ids
        [tokens][used] as `moe_route` leaves them."""
        torch = _torch()
        if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or tuple(prob.shape) != (x.shape[0], experts):
            raise ValueError("x [tokens][hidden], ids [tokens][used], prob [tokens][experts]")
        if prob.dtype != torch.float32 or not prob.is_contiguous():
            raise ValueError("prob is float32 without gaps")
        if w_gate_up.k != x.shape[1] or w_down.rows != experts * x.shape[1] or w_gate_up.rows != experts * 2 * w_down.k:
            raise ValueError("w_gate_up is [experts][2 * ffn][hidden] and w_down [experts][hidden][ffn]")
        if ids.shape[1] > experts:
            raise ValueError("more selections than experts")
        if prob.device != self.device:
            raise self._mx4_elsewhere(prob)
        tokens, used = ids.shape
        hidden = x.shape[1]
        if out is not None and (tuple(out.shape) != (tokens, hidden) or not out.is_contiguous() or out.device != self.device):
            raise ValueError("out is [%d][%d] without gaps" % (tokens, hidden))
        order, token_of, offsets = self.moe_order(ids, experts, tokens_dev=tokens_dev)
        feed = self.mx4_quantize(x, rows=token_of)
        act = self.mx4_matmul_grouped(w_gate_up, experts, feed, offsets, y_dtype=x.dtype, epilogue=EPILOGUE_SWIGLU)
        # (rows that no pair has hold what they held; no expert reads them)
        proj = self.mx4_matmul_grouped(w_down, experts, self.mx4_quantize(act), offsets, y_rows=order, y_dtype=torch.float32)
        return self.moe_combine(proj.view(tokens, used, hidden), prob, ids, tokens_dev=tokens_dev, out=out, out_dtype=out_dtype)
