// See paged_kv.hpp. Behaviour follows compiler/runtime/paged_kv.cpp:10-127.
#include "paged_kv.hpp"

#include <cuda_runtime.h>

#include <algorithm>

#include "ctx.hpp"

namespace mlcb {
namespace runtime {

PagePool::PagePool(uint32_t capacity) : capacity_(capacity), owners_(capacity, 0) {
    stack_.resize(capacity);
    // id 0 ends on top, so a fresh pool allocates in ascending order (paged_kv.cpp:10-17)
    for (uint32_t i = 0; i < capacity; ++i) stack_[i] = capacity - 1 - i;
}

std::optional<uint32_t> PagePool::allocate() {
    if (stack_.empty()) return std::nullopt;
    const uint32_t id = stack_.back();
    stack_.pop_back();
    owners_[id] = 1;
    ++in_use_;
    return id;
}

bool PagePool::allocate_n(size_t n, std::vector<uint32_t>& out) {
    if (n > stack_.size()) return false;
    out.insert(out.end(), stack_.rbegin(), stack_.rbegin() + static_cast<std::ptrdiff_t>(n));
    for (size_t i = out.size() - n; i < out.size(); ++i) owners_[out[i]] = 1;
    stack_.resize(stack_.size() - n);
    in_use_ += n;
    return true;
}

bool PagePool::release(uint32_t page_id) {
    if (page_id >= capacity_ || owners_[page_id] == 0) return false;
    if (owners_[page_id] > 1) {
        --owners_[page_id];
        return true;
    }
    owners_[page_id] = 0;
    stack_.push_back(page_id);
    --in_use_;
    return true;
}

bool PagePool::share(uint32_t page_id) {
    if (page_id >= capacity_ || owners_[page_id] == 0 || owners_[page_id] == UINT32_MAX) return false;
    ++owners_[page_id];
    return true;
}

bool RequestKVState::reserve(PagePool& pool, size_t target_tokens) {
    if (page_size_tokens == 0) return false;
    const size_t needed = (target_tokens + page_size_tokens - 1) / page_size_tokens;
    if (needed <= page_table.size()) return true;  // never shrinks
    return pool.allocate_n(needed - page_table.size(), page_table);
}

bool RequestKVState::fork_from(const RequestKVState& parent, PagePool& pool) {
    if (!page_table.empty() || &parent == this) return false;
    std::vector<uint32_t> table;
    table.reserve(parent.page_table.size());
    for (uint32_t id : parent.page_table) {
        if (!pool.share(id)) {
            for (uint32_t taken : table) pool.release(taken);
            return false;
        }
        table.push_back(id);
    }
    page_table = std::move(table);
    page_size_tokens = parent.page_size_tokens;
    tokens_in_last_page = parent.tokens_in_last_page;
    return true;
}

bool RequestKVState::truncate(PagePool& pool, size_t tokens) {
    if (page_size_tokens == 0 || tokens > total_tokens()) return false;
    const size_t keep = (tokens + page_size_tokens - 1) / page_size_tokens;
    while (page_table.size() > keep) {
        pool.release(page_table.back());
        page_table.pop_back();
    }
    tokens_in_last_page = keep ? static_cast<uint32_t>(tokens - (keep - 1) * page_size_tokens) : 0;
    return true;
}

std::optional<std::pair<uint32_t, uint32_t>> RequestKVState::extend_one_token(PagePool& pool, PageCopies* copies) {
    if (page_size_tokens == 0) return std::nullopt;
    if (!page_table.empty() && tokens_in_last_page < page_size_tokens && pool.owners(page_table.back()) > 1) {
        if (!copies) return std::nullopt;
        copies->reserve(copies->size() + 1);
        const auto id = pool.allocate();
        if (!id) return std::nullopt;  // table unchanged
        copies->emplace_back(page_table.back(), *id);
        pool.release(page_table.back());
        page_table.back() = *id;
    }
    if (page_table.empty() || tokens_in_last_page == page_size_tokens) {
        const auto id = pool.allocate();
        if (!id) return std::nullopt;  // table unchanged
        page_table.push_back(*id);
        tokens_in_last_page = 0;
    }
    return std::make_pair(page_table.back(), tokens_in_last_page++);
}

bool RequestKVState::undo_copy(PagePool& pool, uint32_t from, uint32_t to) {
    const auto at = std::find(page_table.begin(), page_table.end(), to);
    if (at == page_table.end() || !pool.share(from)) return false;
    *at = from;
    pool.release(to);
    return true;
}

std::optional<std::pair<uint32_t, uint32_t>> RequestKVState::locate(size_t pos) const {
    if (page_size_tokens == 0 || pos >= total_tokens()) return std::nullopt;
    return std::make_pair(page_table[pos / page_size_tokens], static_cast<uint32_t>(pos % page_size_tokens));
}

void RequestKVState::release_all(PagePool& pool) {
    for (uint32_t id : page_table) pool.release(id);
    page_table.clear();
    tokens_in_last_page = 0;
}

PagedKVStorage::PagedKVStorage(mlc_ctx* ctx, uint32_t capacity_pages, uint32_t n_layers,
                               uint32_t page_size_tokens, uint32_t n_kv_heads, uint32_t head_dim,
                               uint32_t dtype_bytes)
    : ctx_(ctx), capacity_pages_(capacity_pages), n_layers_(n_layers), page_size_tokens_(page_size_tokens),
      n_kv_heads_(n_kv_heads), head_dim_(head_dim), dtype_bytes_(dtype_bytes),
      k_(n_layers, nullptr), v_(n_layers, nullptr) {}

PagedKVStorage::~PagedKVStorage() {
    if (!ctx_) return;
    for (void* b : k_) if (b) mlc_free(ctx_, b);
    for (void* b : v_) if (b) mlc_free(ctx_, b);
}

bool PagedKVStorage::initialize() {
    if (!ctx_ || !mlc_ctx_available(ctx_)) return false;
    const size_t bytes = static_cast<size_t>(capacity_pages_) * page_bytes();
    if (bytes == 0) return false;
    DeviceGuard guard(ctx_->device);
    for (uint32_t layer = 0; layer < n_layers_; ++layer) {
        if (!k_[layer]) k_[layer] = mlc_alloc(ctx_, bytes);
        if (!v_[layer]) v_[layer] = mlc_alloc(ctx_, bytes);
        if (!k_[layer] || !v_[layer]) return false;
        // unread slots stay zero, like the reference's zero upload (paged_kv.cpp:112-117)
        if (cudaMemsetAsync(k_[layer], 0, bytes, ctx_->stream) != cudaSuccess) return false;
        if (cudaMemsetAsync(v_[layer], 0, bytes, ctx_->stream) != cudaSuccess) return false;
    }
    return cudaStreamSynchronize(ctx_->stream) == cudaSuccess;
}

}  // namespace runtime
}  // namespace mlcb
