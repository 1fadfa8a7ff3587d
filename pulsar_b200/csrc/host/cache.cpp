#include "cache.h"

#include <algorithm>

namespace ph {

FreeList::FreeList(int n) : n_(n), held_(n > 0 ? n : 0, 0) {
    free_.reserve(n > 0 ? n : 0);
    for (int i = n - 1; i >= 0; --i) free_.push_back(i);
}

int FreeList::take() {
    if (free_.empty()) return kOutOfPages;
    const int id = free_.back();
    free_.pop_back();
    held_[id] = 1;
    return id;
}

int FreeList::give(int id) {
    if (id < 0 || id >= n_ || !held_[id]) return kNotHeld;
    held_[id] = 0;
    free_.push_back(id);
    return 0;
}

int Group::take() {
    const int page = pages.take();
    if (page >= 0) holders[page] = 1;
    return page;
}

int Group::share(int page) {
    if (!pages.held(page)) return kNotHeld;
    if (++holders[page] == 2) ++n_shared;
    return 0;
}

int Group::drop(int page) {
    if (!pages.held(page)) return kNotHeld;
    if (--holders[page] == 1) --n_shared;
    return holders[page] > 0 ? 0 : pages.give(page);
}

Cache::Cache(int n_groups, const int* windows, const int* pages, int page_size, int max_requests)
    : page_size_(page_size), slots_(max_requests) {
    groups_.reserve(n_groups);
    for (int g = 0; g < n_groups; ++g) {
        groups_.push_back(Group{windows[g], FreeList(pages[g])});
        groups_.back().holders.assign(pages[g], 0);
        if (windows[g] > 0) windowed_ = true;
    }
}

int Cache::set_keep(int group, int keep_first) {
    if (group < 0 || group >= n_groups() || keep_first < 0 || !reqs_.empty()) return kBadArgument;
    groups_[group].keep = keep_first;
    return 0;
}

const Request* Cache::find(int64_t rid) const {
    auto it = reqs_.find(rid);
    return it == reqs_.end() ? nullptr : &it->second;
}
Request* Cache::find(int64_t rid) {
    auto it = reqs_.find(rid);
    return it == reqs_.end() ? nullptr : &it->second;
}

int Cache::open(int64_t rid) {
    if (reqs_.count(rid)) return kAlreadyOpen;
    const int slot = slots_.take();
    if (slot < 0) return kOutOfSlots;
    Request r;
    r.slot = slot;
    r.tables.resize(groups_.size());
    r.released.resize(groups_.size());
    for (int g = 0; g < n_groups(); ++g) r.released[g] = kept_pages(g);       // the release starts behind the kept pages
    r.synced.assign(groups_.size(), 0);
    reqs_.emplace(rid, std::move(r));
    return slot;
}

void Cache::set_resident_tables(bool on) {
    resident_tables_ = on;
    for (auto& kv : reqs_) kv.second.synced.assign(groups_.size(), 0);      // nothing is known to be on the device
}

// Logical pages below this hold only keys that no query at position >= length sees.
int Cache::first_needed_page(const Group& g, int length) const {
    if (g.window <= 0) return 0;
    const int first_key = length - g.window + 1;          // oldest key the query at `length` sees
    return std::max(0, first_key) / page_size_;
}

int Cache::pages_to_append(const Request& r, int n_new, int group) const {
    const int have = (int)r.tables[group].size();
    const int need = (r.length + n_new + page_size_ - 1) / page_size_;
    return std::max(0, need - have);
}

int Cache::reclaimable(const Request& r, int group) const {
    const int upto = std::min(first_needed_page(groups_[group], r.length), (int)r.tables[group].size());
    int n = 0;                                            // a page that others hold does not become free
    for (int lp = r.released[group]; lp < upto; ++lp) n += groups_[group].holders[r.tables[group][lp]] == 1;
    return n;
}

bool Cache::can_append(const Request& r, int n_new) const {
    for (int g = 0; g < n_groups(); ++g)
        if (pages_to_append(r, n_new, g) > groups_[g].pages.n_free() + reclaimable(r, g)) return false;
    return true;
}

bool Cache::can_admit(int n_tokens) const {
    const int pages = (n_tokens + page_size_ - 1) / page_size_;
    if (slots_.n_free() <= 0) return false;
    for (const Group& g : groups_)
        if (pages > g.pages.n_free()) return false;
    return true;
}

int Cache::release_passed(Request& r) {
    if (!windowed_) return 0;
    int n = 0;
    for (int g = 0; g < n_groups(); ++g) {
        std::vector<int>& table = r.tables[g];
        const int upto = std::min(first_needed_page(groups_[g], r.length), (int)table.size());
        for (int lp = r.released[g]; lp < upto; ++lp) {
            if (groups_[g].drop(table[lp]) != 0) return kNotHeld;
            table[lp] = -1;
            ++n;
        }
        r.released[g] = std::max(r.released[g], upto);
    }
    return n;
}

int Cache::append(int64_t rid, int n_new) {
    if (n_new <= 0) return kBadArgument;
    Request* r = find(rid);
    if (!r) return kUnknownRequest;
    if (!can_append(*r, n_new)) return kOutOfPages;        // either every group gets its pages or nothing changes
    const int rc = release_passed(*r);
    if (rc < 0) return rc;
    for (int g = 0; g < n_groups(); ++g) {
        const int need = pages_to_append(*r, n_new, g);
        for (int i = 0; i < need; ++i) r->tables[g].push_back(groups_[g].take());
    }
    const int start = r->length;
    r->length += n_new;
    return start;
}

int Cache::close(int64_t rid) {
    auto it = reqs_.find(rid);
    if (it == reqs_.end()) return kUnknownRequest;
    Request& r = it->second;
    int rc = 0;
    for (int g = 0; g < n_groups(); ++g)
        for (int page : r.tables[g])
            if (page >= 0 && groups_[g].drop(page) != 0) rc = kNotHeld;
    if (slots_.give(r.slot) != 0) rc = kNotHeld;
    reqs_.erase(it);
    return rc;
}

int Cache::fork(int64_t parent, int64_t child, int length, int* copies) {
    const Request* p = find(parent);
    if (!p) return kUnknownRequest;
    if (has(child)) return kAlreadyOpen;
    if (length < 0 || length > p->length) return kBadArgument;
    const int whole = length / page_size_, rest = length % page_size_;
    for (int g = 0; g < n_groups(); ++g) {
        // what a query at `length` sees has to be there: pages behind a window may have been given back by the parent's later queries
        const int kept = kept_pages(g);
        for (int lp = 0; lp < whole + (rest ? 1 : 0); ++lp)
            if (p->tables[g][lp] < 0 && (lp < kept || lp >= first_needed_page(groups_[g], length))) return kReleasedPage;
        if (rest && groups_[g].pages.n_free() < 1) return kOutOfPages;
    }
    if (slots_.n_free() < 1) return kOutOfSlots;
    const int slot = open(child);
    if (slot < 0) return slot;
    p = find(parent);                                     // (the map has grown)
    Request* c = find(child);
    c->length = length;
    for (int g = 0; g < n_groups(); ++g) {
        std::vector<int>& table = c->tables[g];
        table.assign(p->tables[g].begin(), p->tables[g].begin() + whole);
        for (int page : table)
            if (page >= 0) groups_[g].share(page);
        copies[2 * g] = copies[2 * g + 1] = -1;
        if (rest) {
            table.push_back(groups_[g].take());
            copies[2 * g] = p->tables[g][whole];
            copies[2 * g + 1] = table.back();
        }
        // pages that the parent gave back are none of the child's either
        c->released[g] = std::max(c->released[g], std::min(p->released[g], whole));
    }
    return slot;
}

int Cache::resize(int group, int n_pages, int* from) {
    if (group < 0 || group >= n_groups() || n_pages <= 0) return kBadArgument;
    Group& g = groups_[group];
    const int held = g.pages.n() - g.pages.n_free();
    if (held > n_pages) return kOutOfPages;
    std::vector<int> now(g.pages.n(), -1), holders(n_pages, 0);
    FreeList pages(n_pages);                              // a fresh one yields 0, 1, 2, ...
    for (int page = 0; page < g.pages.n(); ++page) {
        if (!g.pages.held(page)) continue;
        now[page] = pages.take();
        from[now[page]] = page;
        holders[now[page]] = g.holders[page];
    }
    for (auto& kv : reqs_) {
        for (int& page : kv.second.tables[group])
            if (page >= 0) page = now[page];
        kv.second.synced[group] = 0;                      // the device knows the old ids
    }
    g.pages = std::move(pages);
    g.holders = std::move(holders);
    return held;
}

// Every page is free or has as many holders as requests name it; every slot is free or held by exactly one request.
int Cache::check() const {
    for (int g = 0; g < n_groups(); ++g) {
        const Group& group = groups_[g];
        std::vector<int> seen(group.pages.n(), 0);
        int count = 0, shared = 0;
        for (const auto& kv : reqs_)
            for (int page : kv.second.tables[g]) {
                if (page < 0) continue;
                if (page >= group.pages.n() || !group.pages.held(page)) return kInconsistent;
                if (++seen[page] == 1) ++count;
                if (seen[page] == 2) ++shared;
            }
        if (count + group.pages.n_free() != group.pages.n()) return kInconsistent;      // a page was lost
        if (shared != group.n_shared) return kInconsistent;
        for (int page = 0; page < group.pages.n(); ++page)
            if (seen[page] != (group.pages.held(page) ? group.holders[page] : 0)) return kInconsistent;
    }
    std::vector<uint8_t> seen(slots_.n(), 0);
    int count = 0;
    for (const auto& kv : reqs_) {
        const int s = kv.second.slot;
        if (s < 0 || s >= slots_.n() || seen[s] || !slots_.held(s)) return kInconsistent;
        seen[s] = 1;
        ++count;
    }
    return count + slots_.n_free() == slots_.n() ? 0 : kInconsistent;
}

}  // namespace ph
