"""MX4 tensors and the products over them (include/aotx_mx4_b200.h), as methods of `Q8Context`.

An MX4 tensor is rows of k values in blocks of 32 that share a scale, a power of two; a value is one of 0, 0.5, 1, 1.5, 2, 3,
4, 6 with a sign, times the scale of its block: 4.25 bits a value, multiplied by the tensor cores as they are.  Weights are
laid out once with `mx4_quantize` (of a model file's rows: `dequant` gives them as binary16); activations with the
same call or, `mx4_linear`, on their way into a product.

Every method enqueues on the current CUDA stream of PyTorch for the context's device and returns without synchronising.  Like
the rest of the context's methods they are for one thread at a time; tensors used on several streams are ordered by the caller.
"""
EPILOGUE_STORE, EPILOGUE_ADD, EPILOGUE_SWIGLU = 0, 1, 2


def _torch():
    import torch
    return torch


class Mx4Tensor:
    """`rows` rows of k values: codes uint8 [rows][k / 2] (value 2i in the low four bits of byte i), scales uint8
    [ceil(k / 128)][rows][4] (byte b of (c, r): values 128c + 32b .. of row r, 2^(byte - 127); 255 is NaN; 0 past k)."""
    __slots__ = ("codes", "scales", "rows", "k")

    def __init__(self, codes, scales):
        torch = _torch()
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError("codes and scales are uint8, codes [rows][k / 2]")
        self.rows, self.k = codes.shape[0], 2 * codes.shape[1]
        if self.k == 0 or self.k % 32 != 0 or tuple(scales.shape) != ((self.k + 127) // 128, self.rows, 4):
            raise ValueError("k is a multiple of 32 and scales are [ceil(k / 128)][rows][4]")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device:
            raise ValueError("codes and scales lie without gaps on one device")
        self.codes, self.scales = codes, scales

    @classmethod
    def empty(cls, rows, k, device):
        torch = _torch()
        if k <= 0 or k % 32 != 0 or rows < 0:
            raise ValueError("k is a multiple of 32")
        return cls(torch.empty((rows, k // 2), dtype=torch.uint8, device=device),
                   torch.empty(((k + 127) // 128, rows, 4), dtype=torch.uint8, device=device))


def _pointer(t):
    return t.data_ptr() if t is not None else None


class Mx4Calls:
    """The part of Q8Context that works on MX4 tensors."""

    def _mx4_here(self, *tensors):
        for t in tensors:
            if t is not None and t.device != self.device:
                raise ValueError("a tensor on %s, a context for %s" % (t.device, self.device))

    def _mx4_words(self, what, t, count=None):
        """A device array of 32-bit whole numbers."""
        torch = _torch()
        if t is None:
            return
        if t.dtype not in (torch.int32, torch.uint32) or not t.is_contiguous():
            raise ValueError("%s is int32 or uint32 without gaps" % what)
        if count is not None and t.numel() != count:
            raise ValueError("%s has %d entries, not %d" % (what, t.numel(), count))

    def _mx4_code(self, dtype):
        from .q8 import _dtype_code
        try:
            return _dtype_code(dtype)
        except KeyError:
            raise ValueError("float32, float16 or bfloat16, not %s" % dtype) from None

    def _mx4_rows_in(self, x):
        """Rows of 16- or 32-bit values: the type's code and the distance of rows."""
        code = self._mx4_code(x.dtype)
        if x.dim() != 2 or x.shape[1] == 0 or x.shape[1] % 32 != 0:
            raise ValueError("x is [rows][k], k a multiple of 32")
        if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
            raise ValueError("the values of a row lie side by side and rows do not overlap")
        return code, max(x.stride(0), x.shape[1])

    def _mx4_result(self, y, shape, y_dtype, epilogue):
        torch = _torch()
        if epilogue not in (EPILOGUE_STORE, EPILOGUE_ADD, EPILOGUE_SWIGLU):
            raise ValueError("unknown epilogue")
        if y is None:
            if epilogue == EPILOGUE_ADD:
                raise ValueError("EPILOGUE_ADD adds into a y that the caller gives")
            return torch.empty(shape, dtype=y_dtype or torch.float32, device=self.device)
        if tuple(y.shape) != shape or not y.is_contiguous() or (y_dtype is not None and y.dtype != y_dtype):
            raise ValueError("y is %s without gaps" % (shape,))
        self._mx4_here(y)
        return y

    def _mx4_width(self, n, epilogue):
        if epilogue == EPILOGUE_SWIGLU:
            if n % 2 != 0:
                raise ValueError("gate and up rows come in pairs")
            return n // 2
        return n

    # -- quantisation -----------------------------------------------------------------------------------------------
    def mx4_quantize(self, x, rows=None, rows_dev=None, out=None):
        """Rows of x (float32, float16, bfloat16; rows may lie apart) as an Mx4Tensor.  `rows`: int32 row numbers of x, one
        for each row of the result (a number outside x leaves its row as it was).  `rows_dev`: device word with the
        live number of rows."""
        code, stride = self._mx4_rows_in(x)
        self._mx4_words("rows", rows)
        self._mx4_words("rows_dev", rows_dev, 1)
        self._mx4_here(x, rows, rows_dev)
        count = x.shape[0] if rows is None else rows.numel()
        if out is None:
            out = Mx4Tensor.empty(count, x.shape[1], self.device)
        elif out.rows != count or out.k != x.shape[1]:
            raise ValueError("out has %d rows of %d values" % (out.rows, out.k))
        self._mx4_here(out.codes)
        self._check(self._mx4_quantize_call(
            self._address, self._stream(), x.data_ptr(), code, x.shape[0], stride, x.shape[1], _pointer(rows), count,
            _pointer(rows_dev), out.codes.data_ptr(), out.scales.data_ptr()))
        return out

    def mx4_dequant(self, t, first_row=0, rows=None, out=None, dtype=None):
        """The values of rows first_row .. first_row + rows of an MX4 tensor, float16 unless `dtype` or `out` says otherwise."""
        torch = _torch()
        rows = t.rows - first_row if rows is None else rows
        if first_row < 0 or rows < 0 or first_row + rows > t.rows:
            raise ValueError("rows %d .. %d of %d" % (first_row, first_row + rows, t.rows))
        if out is None:
            out = torch.empty((rows, t.k), dtype=dtype or torch.float16, device=self.device)
        elif tuple(out.shape) != (rows, t.k) or not out.is_contiguous() or (dtype is not None and out.dtype != dtype):
            raise ValueError("out is [%d][%d] without gaps" % (rows, t.k))
        code = self._mx4_code(out.dtype)
        self._mx4_here(t.codes, out)
        self._check(self._mx4_dequant_call(self._address, self._stream(), t.codes.data_ptr(), t.scales.data_ptr(), t.rows, t.k,
                                           first_row, rows, out.data_ptr(), code))
        return out

    # -- products ---------------------------------------------------------------------------------------------------
    def mx4_matmul(self, w, x, m_dev=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE):
        """y[m][n] = x . w^T for two MX4 tensors; `m_dev`, `y` and `epilogue` as in `matmul_fused`."""
        if w.k != x.k:
            raise ValueError("rows of %d and of %d values" % (w.k, x.k))
        self._mx4_words("m_dev", m_dev, 1)
        y = self._mx4_result(y, (x.rows, self._mx4_width(w.rows, epilogue)), y_dtype, epilogue)
        self._mx4_here(w.codes, x.codes, m_dev)
        self._check(self._mx4_matmul_call(
            self._address, self._stream(), w.codes.data_ptr(), w.scales.data_ptr(), w.rows, w.k, x.codes.data_ptr(),
            x.scales.data_ptr(), x.rows, _pointer(m_dev), y.data_ptr(), self._mx4_code(y.dtype), epilogue))
        return y

    def mx4_linear(self, w, x, m_dev=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE, workspace=None):
        """`mx4_matmul` of w with `mx4_quantize(x)`, the same y bit for bit; few rows are quantised by the kernel that
        multiplies them."""
        code, stride = self._mx4_rows_in(x)
        m, k = x.shape
        if w.k != k:
            raise ValueError("rows of %d and of %d values" % (w.k, k))
        self._mx4_words("m_dev", m_dev, 1)
        y = self._mx4_result(y, (m, self._mx4_width(w.rows, epilogue)), y_dtype, epilogue)
        self._mx4_here(w.codes, x, m_dev, workspace)
        size = self.lib.aotx_mx4_linear_workspace_bytes(m, k)
        if workspace is None:
            if size:
                torch = _torch()
                workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
        else:
            size = workspace.numel() * workspace.element_size()
            if not workspace.is_contiguous():
                raise ValueError("the workspace has gaps")
        self._check(self._mx4_linear_call(
            self._address, self._stream(), w.codes.data_ptr(), w.scales.data_ptr(), w.rows, k, x.data_ptr(), code, stride, m,
            _pointer(m_dev), y.data_ptr(), self._mx4_code(y.dtype), epilogue, _pointer(workspace), size))
        return y

    # -- routed experts ---------------------------------------------------------------------------------------------
    def moe_order(self, ids, experts, tokens_dev=None):
        """The (token, rank) pairs of ids [tokens][used] by expert: order (the pair at each place), their tokens, and
        offsets [experts + 1] of the experts' places; int32, places that no pair has hold -1."""
        torch = _torch()
        self._mx4_words("ids", ids)
        self._mx4_words("tokens_dev", tokens_dev, 1)
        if ids.dim() != 2 or ids.shape[1] == 0:
            raise ValueError("ids is [tokens][used]")
        self._mx4_here(ids, tokens_dev)
        tokens, used = ids.shape
        order = torch.empty(tokens * used, dtype=torch.int32, device=self.device)
        token_of = torch.empty(tokens * used, dtype=torch.int32, device=self.device)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=self.device)
        self._check(self._mx4_order_call(self._address, self._stream(), ids.data_ptr(), tokens, _pointer(tokens_dev), used,
                                         experts, order.data_ptr(), token_of.data_ptr(), offsets.data_ptr()))
        return order, token_of, offsets

    def mx4_matmul_grouped(self, w, experts, x, offsets, y_rows=None, y=None, y_dtype=None, epilogue=EPILOGUE_STORE):
        """Rows offsets[e] .. offsets[e + 1] of x times expert e's rows of w (w.rows / experts each).  `y_rows`: int32, the row
        of y for each row of x (one outside y is left out).  Rows that no expert has are not written."""
        if w.k != x.k:
            raise ValueError("rows of %d and of %d values" % (w.k, x.k))
        if experts <= 0 or w.rows % experts != 0:
            raise ValueError("%d rows of w for %d experts" % (w.rows, experts))
        if epilogue == EPILOGUE_ADD:
            raise ValueError("grouped products store or apply the gated unit")
        self._mx4_words("offsets", offsets, experts + 1)
        self._mx4_words("y_rows", y_rows, x.rows)
        n = w.rows // experts
        width = self._mx4_width(n, epilogue)
        if y is not None and y.dim() != 2:
            raise ValueError("y is [rows][%d]" % width)
        rows = x.rows if y is None or y_rows is None else y.shape[0]
        y = self._mx4_result(y, (rows, width), y_dtype, epilogue)
        self._mx4_here(w.codes, x.codes, offsets, y_rows)
        self._check(self._mx4_grouped_call(
            self._address, self._stream(), w.codes.data_ptr(), w.scales.data_ptr(), experts, n, w.k, x.codes.data_ptr(),
            x.scales.data_ptr(), x.rows, offsets.data_ptr(), _pointer(y_rows), rows, y.data_ptr(),
            self._mx4_code(y.dtype), epilogue))
        return y

    def mx4_moe_ffn(self, w_gate_up, w_down, experts, x, prob, ids, tokens_dev=None, out=None, out_dtype=None):
        """The routed feed-forward step of `moe_ffn_fused` on MX4 weights (gate and up rows of an expert interleaved): the
        pairs in the experts' order, their rows of x quantised, gate and up by expert with the gated unit, its binary16
        result quantised, the down product by expert, and the rank-ordered weighted sum.  x is any type that
        `mx4_quantize` takes; prob [tokens][experts] float32 and ids [tokens][used] as `moe_route` leaves them."""
        torch = _torch()
        if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or tuple(prob.shape) != (x.shape[0], experts):
            raise ValueError("x [tokens][hidden], ids [tokens][used], prob [tokens][experts]")
        if prob.dtype != torch.float32 or not prob.is_contiguous():
            raise ValueError("prob is float32 without gaps")
        if w_gate_up.k != x.shape[1] or w_down.rows != experts * x.shape[1] or w_gate_up.rows != experts * 2 * w_down.k:
            raise ValueError("w_gate_up is [experts][2 * ffn][hidden] and w_down [experts][hidden][ffn]")
        if ids.shape[1] > experts:
            raise ValueError("more selections than experts")
        self._mx4_here(prob)
        tokens, used = ids.shape
        hidden = x.shape[1]
        order, token_of, offsets = self.moe_order(ids, experts, tokens_dev=tokens_dev)
        feed = self.mx4_quantize(x, rows=token_of)
        act = self.mx4_matmul_grouped(w_gate_up, experts, feed, offsets, y_dtype=torch.float16, epilogue=EPILOGUE_SWIGLU)
        # (rows that no pair has hold what they held; no expert reads them)
        proj = self.mx4_matmul_grouped(w_down, experts, self.mx4_quantize(act), offsets, y_rows=order, y_dtype=torch.float32)
        return self.moe_combine(proj.view(tokens, used, hidden), prob, ids, tokens_dev=tokens_dev, out=out, out_dtype=out_dtype)
