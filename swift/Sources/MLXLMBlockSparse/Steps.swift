import CBSAttn
import MLX

/// New tokens of up to 64 requests in a model's layers, each request with its
/// own number of them, as a tree of drafts or as a chain: the general form of
/// SpeculativeTokenIterator.speculateRound (Evaluate.swift:841-931).  Packed
/// tensors are [rows, heads, D]; request i's tokens are its rows starts[i] ..<
/// starts[i] + taken[i].  `map` once for all layers, then for each layer
/// `appendPacked`, `attendTree` and, once the accepted paths are known, `keep`.
/// Nothing in it waits for the host.  One stream at a time; keep the object
/// while calls that use it are pending.
public final class BlockSparseStep {
    public let caches: [BlockSparseKVCache]
    public let rows: Int
    public let maxTokens: Int
    /// Written by `map`, on the device: [64 + 1], [64], [rows], [rows], [rows]
    /// (nil where maxTokens > 64), [caches, rows] and [caches * 64] of which
    /// the first n (+ 1), n and caches * n entries of the per-request ones hold.
    public let starts, taken, requests, positions, slots, ends: MLXArray
    public let ancestors: MLXArray?
    /// One place for the object's life: the library knows a captured step by it.
    let step = UnsafeMutablePointer<bsattn_step>.allocate(capacity: 1)

    public init(caches: [BlockSparseKVCache], rows: Int, maxTokens: Int) {
        precondition(caches.count >= 1 && caches.count <= Int(BSATTN_STEP_CACHES) && rows >= 1 && maxTokens >= 1,
                     "a step takes 1 to 128 caches, and at least a row and a token")
        self.caches = caches
        self.rows = rows
        self.maxTokens = maxTokens
        let device = caches[0].device
        let most = Int(BSATTN_STEP_SEQS)
        func new(_ shape: [Int]) -> MLXArray { device.empty(shape, dtype: .int32) }
        starts = new([most + 1])
        taken = new([most])
        requests = new([rows])
        positions = new([rows])
        slots = new([caches.count, rows])
        ends = new([caches.count * most])
        ancestors = maxTokens <= Int(BSATTN_TREE_NODES) ? device.empty([rows], dtype: .uint64) : nil
        func at(_ x: MLXArray) -> UnsafeMutablePointer<Int32> { device.pointer(x).assumingMemoryBound(to: Int32.self) }
        step.initialize(to: .init())
        step.pointee.n_caches = Int32(caches.count)
        step.pointee.rows = Int32(rows)
        step.pointee.max_tokens = Int32(maxTokens)
        step.pointee.starts = at(starts)
        step.pointee.taken = at(taken)
        step.pointee.requests = at(requests)
        step.pointee.positions = at(positions)
        step.pointee.ancestors = ancestors.map { device.pointer($0).assumingMemoryBound(to: UInt64.self) }
        step.pointee.slots = at(slots)
        step.pointee.ends = at(ends)
    }

    deinit { step.deallocate() }

    /// counts [n] int32: tokens of each request, whose pages are held already
    /// (reserve); parents [rows] int32: each node's parent among its request's
    /// tokens, or -1 (nil: chains).
    public func map(counts: MLXArray, parents: MLXArray? = nil, seqIds: [Int]? = nil) {
        precondition(counts.ndim == 1 && counts.dtype == .int32, "counts must be [n] int32")
        precondition(parents == nil || (parents!.shape == [rows] && parents!.dtype == .int32), "parents must be [rows] int32")
        let device = caches[0].device
        func at(_ x: MLXArray) -> UnsafePointer<Int32> {
            UnsafePointer(device.pointer(x).assumingMemoryBound(to: Int32.self))
        }
        let handles: [OpaquePointer?] = caches.map { $0.handle }
        let (c, p) = (at(counts), parents.map(at))
        withSeqIds(seqIds, rows: counts.dim(0)) { ids in
            handles.withUnsafeBufferPointer { h in
                bsCheck(bsattn_step_map(h.baseAddress, step, c, p, ids, Int32(counts.dim(0)), caches[0].stream),
                        "bsattn_step_map")
            }
        }
    }
}

extension BlockSparseKVCache {
    /// Takes the pages for n more tokens of each listed sequence now, so that
    /// steps need no host work.
    public func reserve(_ n: Int, seqIds: [Int]) {
        withSeqIds(seqIds, rows: seqIds.count) { ids in
            bsCheck(bsattn_reserve(handle, ids, Int32(seqIds.count), Int32(n), stream), "bsattn_reserve")
        }
    }

    /// Copies the device-side lengths back, behind which the host's view is
    /// after a step.  Waits for the stream.
    public func sync() {
        bsCheck(bsattn_sync(handle, stream), "bsattn_sync")
    }

    func checkPacked(_ x: MLXArray, _ step: BlockSparseStep, heads: Int) {
        precondition(x.shape == [step.rows, heads, headDim] && x.dtype == dtype, "packed tensors must be [rows, heads, D] in the cache's dtype")
    }

    /// Appends a step's rows, keys and values [rows, Hkv, D], where its map put them.
    public func appendPacked(keys: MLXArray, values: MLXArray, step: BlockSparseStep) {
        checkPacked(keys, step, heads: kvHeads)
        checkPacked(values, step, heads: kvHeads)
        bsCheck(bsattn_append_packed(handle, step.step, device.pointer(keys), nil, device.pointer(values), nil, stream),
                "bsattn_append_packed")
    }

    /// Dense attention of a step's rows, queries [rows, Hq, D], after their
    /// append and before `keep`: each sees what its request held before and its
    /// ancestors in the tree, or those at the last `window` positions.  Rows of
    /// no request are undefined.
    public func attendTree(queries: MLXArray, step: BlockSparseStep, scale: Float, window: Int? = nil,
                           sinks: MLXArray? = nil) -> MLXArray
    {
        checkPacked(queries, step, heads: qHeads)
        precondition(window == nil || window! >= 1, "window must be at least 1")
        precondition(sinks == nil || (sinks!.shape == [qHeads] && sinks!.dtype == .float32),
                     "sinks must be [Hq] float32")
        let out = device.empty(queries.shape, dtype: dtype)
        let sp = sinks.map { UnsafePointer(device.pointer($0).assumingMemoryBound(to: Float.self)) }
        bsCheck(bsattn_attend_tree(handle, step.step, device.pointer(queries), nil, Int32(window ?? 0), sp, scale,
                                   device.pointer(out), stream), "bsattn_attend_tree")
        return out
    }

    /// Of the tokens that the step appended, request i keeps its nodes kept[i,
    /// ..< nKept[i]] (int32 [n, width] and [n], ascending), moved together
    /// behind what it held before.  Once nodes have moved, only a keep of none
    /// (or `appendPacked` again) finds the step's.
    public func keep(step: BlockSparseStep, kept: MLXArray, nKept: MLXArray) {
        precondition(kept.ndim == 2 && kept.dim(1) >= 1 && kept.dtype == .int32 && nKept.shape == [kept.dim(0)]
                         && nKept.dtype == .int32 && kept.dim(0) == Int(step.step.pointee.n_seqs),
                     "kept must be [n, width] and nKept [n], int32")
        func at(_ x: MLXArray) -> UnsafePointer<Int32> {
            UnsafePointer(device.pointer(x).assumingMemoryBound(to: Int32.self))
        }
        bsCheck(bsattn_keep(handle, step.step, at(kept), Int32(kept.dim(1)), at(nKept), stream), "bsattn_keep")
    }
}
