import CBSAttn
import MLX

/// Rotary positions of the first `dims` dims of each head, as the kernels take
/// them: radians per position of every pair (64-bit) and a factor on the
/// rotated dims.  The variants that RoPEUtils.swift:210 chooses from a model's
/// rope_scaling entry differ in these two only.  Keep the object while calls
/// that use it are pending.
public final class BlockSparseRoPE {
    let table: MLXArray  // the angles' words, little-endian
    let device: BlockSparseDevice
    public let dims: Int
    public let traditional: Bool
    public let factor: Float

    /// `theta`: dims / 2 angles.  `traditional`: pairs are neighbours
    /// (2i, 2i + 1), otherwise (i, i + dims / 2).
    public init(dims: Int, traditional: Bool, theta: [Double], factor: Float = 1, device: BlockSparseDevice) {
        precondition(dims >= 2 && dims % 2 == 0 && theta.count == dims / 2, "rope theta must hold dims / 2 angles")
        self.dims = dims
        self.traditional = traditional
        self.factor = factor
        self.device = device
        self.table = MLXArray(theta.flatMap { t -> [UInt32] in
            let bits = t.bitPattern
            return [UInt32(truncatingIfNeeded: bits), UInt32(truncatingIfNeeded: bits >> 32)]
        })
    }

    var angles: bsattn_rope {
        .init(theta: UnsafePointer(device.pointer(table).assumingMemoryBound(to: Double.self)), dims: Int32(dims),
              interleaved: traditional ? 1 : 0, factor: factor, reserved: 0)
    }
}

extension BlockSparseKVCache {
    /// Dense decode: attention of queries [B, Hq, 1, D] over every token of
    /// the sequences (the new one appended), or over the last `window`, for
    /// layers that take no block selection.  `sinks`: [Hq] float32 logits that
    /// join each head's softmax without a value.
    public func decodeDense(queries: MLXArray, scale: Float, window: Int? = nil, sinks: MLXArray? = nil,
                            seqIds: [Int]? = nil) -> MLXArray
    {
        checkQueries(queries)
        precondition(window == nil || window! >= 1, "window must be at least 1")
        precondition(sinks == nil || (sinks!.shape == [qHeads] && sinks!.dtype == .float32),
                     "sinks must be [Hq] float32")
        let out = device.empty(queries.shape, dtype: dtype)
        let (qp, op) = (device.pointer(queries), device.pointer(out))
        let sp = sinks.map { UnsafePointer(device.pointer($0).assumingMemoryBound(to: Float.self)) }
        withSeqIds(seqIds, rows: queries.dim(0)) { ids in
            bsCheck(bsattn_decode_dense(handle, qp, ids, Int32(queries.dim(0)), Int32(window ?? 0), sp, scale, op,
                                        stream), "bsattn_decode_dense")
        }
        return out
    }

    /// Sequence dst[i] (empty) becomes the first tokens[i] tokens of src[i]
    /// (default: all of them): full blocks are shared, a partial last block is
    /// copied, and the sequences are independent from then on.
    public func fork(_ src: [Int], to dst: [Int], tokens: [Int]? = nil) {
        precondition(src.count == dst.count && (tokens == nil || tokens!.count == src.count),
                     "src, dst and tokens must have one entry per fork")
        withSeqIds(src, rows: src.count) { from in
            withSeqIds(dst, rows: src.count) { to in
                withSeqIds(tokens, rows: src.count) { n in
                    bsCheck(bsattn_fork(handle, from, to, Int32(src.count), n, stream), "bsattn_fork")
                }
            }
        }
    }

    /// applyRotaryPosition (RoPEApplication.swift:23-27): x [B, H, L, D] at the
    /// positions that follow the cached tokens, or at `positions` [B, L] int32.
    public func applyRotaryPosition(_ rope: BlockSparseRoPE, to x: MLXArray, positions: MLXArray? = nil,
                                    seqIds: [Int]? = nil) -> MLXArray
    {
        precondition(x.ndim == 4 && x.dim(3) == headDim && x.dtype == dtype, "x must be [B, H, L, D] in the cache's dtype")
        let pos = positionsPointer(positions, shape: [x.dim(0), x.dim(2)])
        let out = device.empty(x.shape, dtype: dtype)
        let (xp, op) = (device.pointer(x), device.pointer(out))
        var angles = rope.angles
        withSeqIds(seqIds, rows: x.dim(0)) { ids in
            bsCheck(bsattn_rotate(handle, &angles, xp, nil, Int32(x.dim(1)), ids, Int32(x.dim(0)), Int32(x.dim(2)),
                                  pos, op, stream), "bsattn_rotate")
        }
        return out
    }

    /// RMS norms of the heads of queries [B, Hq, L, D] and keys [B, Hkv, L, D]
    /// (weights [D], both nil: none), then their positions, in one pass.
    public func normRotate(_ rope: BlockSparseRoPE, queries: MLXArray, keys: MLXArray, qWeight: MLXArray?,
                           kWeight: MLXArray?, eps: Float, weightOffset: Float = 0, positions: MLXArray? = nil,
                           seqIds: [Int]? = nil) -> (MLXArray, MLXArray)
    {
        checkQueries(queries, multi: true)
        precondition(keys.shape == [queries.dim(0), kvHeads, queries.dim(2), headDim] && keys.dtype == dtype,
                     "keys must be [B, Hkv, L, D] in the cache's dtype")
        for w in [qWeight, kWeight] {
            precondition(w == nil || (w!.shape == [headDim] && w!.dtype == dtype), "norm weights must be [D] in the cache's dtype")
        }
        let pos = positionsPointer(positions, shape: [queries.dim(0), queries.dim(2)])
        let q = device.empty(queries.shape, dtype: dtype)
        let k = device.empty(keys.shape, dtype: dtype)
        let (qp, kp, qo, ko) = (device.pointer(queries), device.pointer(keys), device.pointer(q), device.pointer(k))
        let (qw, kw) = (qWeight.map { device.pointer($0) }, kWeight.map { device.pointer($0) })
        var angles = rope.angles
        withSeqIds(seqIds, rows: queries.dim(0)) { ids in
            bsCheck(bsattn_norm_rotate(handle, &angles, qp, nil, kp, nil, qw, kw, eps, weightOffset, ids,
                                       Int32(queries.dim(0)), Int32(queries.dim(2)), pos, qo, ko, stream),
                    "bsattn_norm_rotate")
        }
        return (q, k)
    }

    func positionsPointer(_ positions: MLXArray?, shape: [Int]) -> UnsafePointer<Int32>? {
        guard let positions else { return nil }
        precondition(positions.dtype == .int32 && positions.shape == shape, "positions must be int32 [B, L]")
        return UnsafePointer(device.pointer(positions).assumingMemoryBound(to: Int32.self))
    }
}
