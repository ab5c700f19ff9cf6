// Page and slot management, the batch step, the continuous-batching scheduler, and their C entry points.
#include "engine.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../ir/module_api.hpp"
#include "capi_types.hpp"

namespace oxrt {

using namespace ox;

namespace {

bool starts_with(const std::string& s, const char* prefix) { return s.rfind(prefix, 0) == 0; }

// splitmix64 (Steele, Lea, Flood: "Fast splittable pseudorandom number generators"): one uniform in [0, 1) per draw
float next_uniform(uint64_t& state) {
    uint64_t z = (state += 0x9E3779B97F4A7C15ull);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    return (float)(z >> 40) * (1.f / 16777216.f);
}

}  // namespace

bool Engine::serves(const Module& m) {
    for (auto& in : m.inputs)
        if (in.first == "seq_info") return true;
    return false;
}

Engine::Engine(Session& s, int64_t max_tokens, int32_t max_seqs) : s_(s), max_seqs_(max_seqs) {
    const Module& m = s.module();
    if (!serves(m)) fail(ErrKind::Binding, "the module has no 'seq_info' input: it does not run ragged batches");
    if (max_tokens <= 0 || max_seqs <= 0) fail(ErrKind::Shape, "an engine needs room for at least one token and one sequence");
    const auto& outs = s.output_names();
    for (size_t o = 0; o < outs.size(); o++)
        if (outs[o] == "logits") logits_out_ = (int)o;
    if (logits_out_ < 0) fail(ErrKind::Binding, "output 'logits' missing");
    const TensorType& lt = m.values[m.outputs[(size_t)logits_out_].second].ty;
    if (lt.dtype != DType::F32 || lt.shape.size() != 2 || !lt.shape[1].as_const()) fail(ErrKind::DType, "output 'logits' must be F32 [num_logits, vocab]");
    vocab_ = (int64_t)*lt.shape[1].as_const();

    for (auto& in : m.inputs) {
        names_.push_back(in.first);
        if (!starts_with(in.first, "pages.") || page_) continue;
        const TensorType& t = m.values[in.second].ty;
        // [num_pages, …, page, …]: key pools carry the page on axis 2, per-token scalars on axis 1
        const size_t axis = t.shape.size() == 2 ? 1 : 2;
        if (t.shape.size() < 2 || !t.shape[axis].as_const()) fail(ErrKind::Shape, "input '" + in.first + "' has no constant page axis");
        page_ = (int64_t)*t.shape[axis].as_const();
    }
    if (!page_) page_ = 64;  // a module without attention keeps no pages; lengths are still counted in them
    n_pages_ = pages_for(max_tokens);
    Bindings b;
    auto bind = [&](const char* name, uint64_t v) {
        if (auto id = m.symbols.get(name)) b.bind(*id, v);
    };
    bind("num_pages", (uint64_t)n_pages_);
    bind("num_slots", (uint64_t)max_seqs);
    state_.resize(names_.size());
    updated_.assign(names_.size(), -1);
    for (size_t i = 0; i < names_.size(); i++) {
        if (!starts_with(names_[i], "pages.") && !starts_with(names_[i], "slots.")) continue;
        const TensorType& t = m.values[m.inputs[i].second].ty;
        std::vector<int64_t> shape;
        for (auto& d : t.shape) shape.push_back((int64_t)d.eval(b));
        state_[i] = s.zeros(t.dtype, shape);
        for (size_t o = 0; o < outs.size(); o++)
            if (outs[o] == "updated." + names_[i]) updated_[i] = (int)o;
        if (updated_[i] < 0) fail(ErrKind::Binding, "output 'updated." + names_[i] + "' missing");
    }
    for (int64_t i = n_pages_; i-- > 0;) free_pages_.push_back((int32_t)i);
    for (int32_t i = max_seqs; i-- > 0;) free_slots_.push_back(i);
}

int64_t Engine::length(int64_t id) const {
    auto it = seqs_.find(id);
    return it == seqs_.end() ? 0 : it->second.past;
}

void Engine::release(int64_t id) {
    auto it = seqs_.find(id);
    if (it == seqs_.end()) fail(ErrKind::Binding, "no live sequence with id " + std::to_string(id));
    // the next owner of these pages and this slot runs behind everything enqueued so far
    for (size_t i = it->second.pages.size(); i-- > 0;) free_pages_.push_back(it->second.pages[i]);
    free_slots_.push_back(it->second.slot);
    seqs_.erase(it);
}

DTensor Engine::forward(const std::vector<Entry>& entries, const DTensor* ids_dev) {
    if (entries.empty()) fail(ErrKind::Shape, "a step needs at least one entry");
    // what the step needs, before anything is taken
    int64_t new_pages = 0, new_slots = 0, rows = 0;
    for (size_t i = 0; i < entries.size(); i++) {
        const Entry& e = entries[i];
        if (e.n_tokens <= 0) fail(ErrKind::Shape, "an entry brings at least one token");
        for (size_t j = 0; j < i; j++)
            if (entries[j].id == e.id) fail(ErrKind::Binding, "sequence " + std::to_string(e.id) + " appears twice in one step");
        for (int32_t w = 0; w < e.n_want; w++)
            if (e.want[w] < 0 || e.want[w] >= e.n_tokens) fail(ErrKind::Shape, "a wanted place lies outside the entry's tokens");
        auto it = seqs_.find(e.id);
        const int64_t past = it == seqs_.end() ? 0 : it->second.past, have = it == seqs_.end() ? 0 : (int64_t)it->second.pages.size();
        if (past + e.n_tokens > INT32_MAX / 2) fail(ErrKind::Shape, "sequence too long");
        new_pages += std::max<int64_t>(0, pages_for(past + e.n_tokens) - have);
        new_slots += it == seqs_.end();
        rows += e.n_tokens;
    }
    if (new_slots > (int64_t)free_slots_.size()) fail(ErrKind::Runtime, "no free slot for a new sequence");
    if (new_pages > (int64_t)free_pages_.size())
        fail(ErrKind::Runtime, "out of cache pages: " + std::to_string(new_pages) + " needed, " + std::to_string(free_pages_.size()) + " free");

    std::vector<int64_t> ids, want;
    std::vector<int32_t> info;
    size_t widest = 1;
    int64_t row = 0;
    for (auto& e : entries) {
        auto it = seqs_.find(e.id);
        if (it == seqs_.end()) {
            it = seqs_.emplace(e.id, Seq{}).first;
            it->second.slot = free_slots_.back();
            free_slots_.pop_back();
        }
        Seq& q = it->second;
        while ((int64_t)q.pages.size() < pages_for(q.past + e.n_tokens)) {
            q.pages.push_back(free_pages_.back());
            free_pages_.pop_back();
        }
        widest = std::max(widest, q.pages.size());
        info.insert(info.end(), {(int32_t)row, e.n_tokens, (int32_t)q.past, q.slot});
        if (!ids_dev) ids.insert(ids.end(), e.tokens, e.tokens + e.n_tokens);
        for (int32_t w = 0; w < e.n_want; w++) want.push_back(row + e.want[w]);
        row += e.n_tokens;
    }
    if (want.empty()) want.push_back(rows - 1);
    // four table widths per power of two: a plan (and its graph) serves a sequence while it grows, and a launch that is
    // sized by the width is not far off
    size_t width = 4;
    for (size_t quarter = 1; width < widest; width += quarter)
        if (width == 8 * quarter) quarter *= 2;
    std::vector<int32_t> table(entries.size() * width, 0);
    for (size_t i = 0; i < entries.size(); i++) {
        const Seq& q = seqs_[entries[i].id];
        std::copy(q.pages.begin(), q.pages.end(), table.begin() + (long)(i * width));
    }
    const int64_t R = (int64_t)entries.size();
    // what describes the step, in one copy
    std::vector<Session::HostPart> parts = {{DType::I32, {R, 4}, info.data(), info.size() * 4},
                                            {DType::I32, {R, (int64_t)width}, table.data(), table.size() * 4},
                                            {DType::I64, {(int64_t)want.size()}, want.data(), want.size() * 8}};
    if (!ids_dev) parts.push_back({DType::I64, {rows}, ids.data(), ids.size() * 8});
    const std::vector<DTensor> step = s_.upload_together(parts);
    std::vector<std::pair<std::string, DTensor>> feed;
    feed.reserve(names_.size());
    for (size_t i = 0; i < names_.size(); i++) {
        const std::string& n = names_[i];
        DTensor t;
        if (n == "input_ids") t = ids_dev ? *ids_dev : step[3];
        else if (n == "seq_info") t = step[0];
        else if (n == "page_table") t = step[1];
        else if (n == "logit_rows") t = step[2];
        else if (state_[i].buf) t = state_[i];
        else fail(ErrKind::Binding, "input '" + n + "' is not one the engine can fill");
        feed.emplace_back(n, std::move(t));
    }
    auto outs = s_.run(feed);
    for (size_t i = 0; i < names_.size(); i++)
        if (updated_[i] >= 0) state_[i] = outs[(size_t)updated_[i]].second;
    for (auto& e : entries) seqs_[e.id].past += e.n_tokens;
    return outs[(size_t)logits_out_].second;
}

// ───────────────────────────── scheduling ───────────────────────────────
int64_t Engine::submit(std::vector<int64_t> prompt, int32_t max_new, int64_t eos, const Sampling& sampling) {
    if (prompt.empty()) fail(ErrKind::Shape, "Cannot prefill with empty input_ids");
    if (max_new <= 0) fail(ErrKind::Shape, "a request generates at least one token");
    Request r;
    r.id = next_request_++;
    r.pages = pages_for((int64_t)prompt.size() + max_new - 1);  // the last token is never run
    if (r.pages > n_pages_) fail(ErrKind::Shape, "the request needs " + std::to_string(r.pages) + " pages, the engine has " + std::to_string(n_pages_));
    r.prompt = std::move(prompt);
    r.left = max_new;
    r.eos = eos;
    r.sampling = sampling;
    r.rng = sampling.seed;
    waiting_.push_back(std::move(r));
    return waiting_.back().id;
}

void Engine::cancel(int64_t request) {
    for (auto it = waiting_.begin(); it != waiting_.end(); ++it)
        if (it->id == request) {
            waiting_.erase(it);
            return;
        }
    for (auto it = running_.begin(); it != running_.end(); ++it)
        if (it->id == request) {
            reserved_ -= it->pages;
            if (seqs_.count(request)) release(request);
            running_.erase(it);
            return;
        }
}

Engine::Request& Engine::request_of(int64_t id) {
    for (auto& r : waiting_)
        if (r.id == id) return r;
    for (auto& r : running_)
        if (r.id == id) return r;
    fail(ErrKind::Binding, "no unfinished request " + std::to_string(id));
}

// What the biases of each token add up to, in their order and in f32 as the kernel does: (token, sum).
static std::vector<std::pair<int32_t, float>> bias_sums(const Engine::Rules& r) {
    std::vector<std::pair<int32_t, float>> sums;
    for (size_t i = 0; i < r.bias.size(); i++) sums.emplace_back(r.bias_ids[i], r.bias[i]);
    std::stable_sort(sums.begin(), sums.end(), [](const auto& a, const auto& b) { return a.first < b.first; });
    size_t n = 0;
    for (size_t i = 0; i < sums.size(); i++) {
        if (n && sums[n - 1].first == sums[i].first) sums[n - 1].second += sums[i].second;
        else sums[n++] = sums[i];
    }
    sums.resize(n);
    return sums;
}

// Whether some token of `vocab` is allowed and has not minus infinity for its biases.
static bool leaves_a_token(const Engine::Rules& r, int64_t vocab) {
    int64_t left = r.allowed.empty() ? vocab : 0;
    for (uint32_t w : r.allowed) left += __builtin_popcount(w);
    for (auto& [token, sum] : bias_sums(r)) left -= sum == -INFINITY && (r.allowed.empty() || (r.allowed[(size_t)token / 32] >> (token % 32) & 1u));
    return left > 0;
}

void Engine::constrain(int64_t request, float repetition, float frequency, float presence, std::vector<int32_t> bias_ids, std::vector<float> bias) {
    Request& r = request_of(request);
    if (!(repetition > 0.f) || !std::isfinite(repetition)) fail(ErrKind::Attribute, "a repetition penalty is a factor above 0");
    if (!std::isfinite(frequency) || !std::isfinite(presence)) fail(ErrKind::Attribute, "penalties must be finite");
    if (bias_ids.size() != bias.size() || (int64_t)bias.size() > kMaxBiases) fail(ErrKind::Shape, "at most " + std::to_string(kMaxBiases) + " biases of a request");
    for (size_t i = 0; i < bias.size(); i++) {
        if (bias_ids[i] < 0 || bias_ids[i] >= vocab_) fail(ErrKind::Shape, "a bias of token " + std::to_string(bias_ids[i]) + ", which is not one of " + std::to_string(vocab_));
        if (std::isnan(bias[i]) || bias[i] == INFINITY) fail(ErrKind::Attribute, "a bias is a number, or minus infinity");
    }
    Rules rules{repetition, frequency, presence, std::move(bias_ids), std::move(bias), r.rules.allowed};
    for (auto& [token, sum] : bias_sums(rules))
        if (sum == INFINITY) fail(ErrKind::Attribute, "the biases of token " + std::to_string(token) + " add up to more than f32 holds");
    if (!leaves_a_token(rules, vocab_)) fail(ErrKind::Shape, "the biases leave no token");
    r.rules = std::move(rules);
}

void Engine::allow(int64_t request, std::vector<uint32_t> allowed) {
    Request& r = request_of(request);
    if (!allowed.empty()) {
        if ((int64_t)allowed.size() != (vocab_ + 31) / 32) fail(ErrKind::Shape, "a mask has a bit for each of " + std::to_string(vocab_) + " tokens");
        if (vocab_ % 32) allowed.back() &= (1u << (vocab_ % 32)) - 1;
        if (std::all_of(allowed.begin(), allowed.end(), [](uint32_t w) { return w == 0; })) fail(ErrKind::Shape, "the mask allows no token");
    }
    allowed.swap(r.rules.allowed);
    if (!leaves_a_token(r.rules, vocab_)) {
        allowed.swap(r.rules.allowed);
        fail(ErrKind::Shape, "the mask and the biases leave no token");
    }
}

// The rows' logits under their requests' rules; those of a batch without any are left alone.
DTensor Engine::constrained(const DTensor& logits, const std::vector<Request*>& rows) {
    const size_t n = rows.size(), words = (size_t)(vocab_ + 31) / 32;
    size_t longest = 0, biases = 0, masks = 0;
    bool any = false;
    for (const Request* r : rows) {
        any = any || r->rules.any();
        if (r->rules.history()) longest = std::max(longest, r->prompt.size() + r->answer.size());
        biases = std::max(biases, r->rules.bias.size());
        masks += !r->rules.allowed.empty();
    }
    if (!any) return logits;
    std::vector<int32_t> history(n * longest), lengths(n * 2), bias_ids(n * biases, -1), mask_of(n, -1);
    std::vector<float> penalties(n * 3), bias(n * biases);
    std::vector<uint32_t> allowed;
    allowed.reserve(masks * words);
    for (size_t i = 0; i < n; i++) {
        const Request& r = *rows[i];
        if (r.rules.history()) {
            // (a prompt may hold tokens that have an embedding and no logit: nothing is to be penalised)
            int32_t *const from = history.data() + i * longest, *at = from;
            for (const std::vector<int64_t>* part : {&r.prompt, &r.answer}) {
                for (int64_t t : *part)
                    if (t >= 0 && t < vocab_) *at++ = (int32_t)t;
                lengths[2 * i + (part == &r.answer)] = (int32_t)(at - from);
            }
        }
        penalties[3 * i] = r.rules.repetition, penalties[3 * i + 1] = r.rules.frequency, penalties[3 * i + 2] = r.rules.presence;
        std::copy(r.rules.bias_ids.begin(), r.rules.bias_ids.end(), bias_ids.begin() + (long)(i * biases));
        std::copy(r.rules.bias.begin(), r.rules.bias.end(), bias.begin() + (long)(i * biases));
        if (!r.rules.allowed.empty()) {
            mask_of[i] = (int32_t)(allowed.size() / words);
            allowed.insert(allowed.end(), r.rules.allowed.begin(), r.rules.allowed.end());
        }
    }
    const int64_t N = (int64_t)n;
    const std::vector<DTensor> t = s_.upload_together({{DType::I32, {N, (int64_t)longest}, history.data(), history.size() * 4},
                                                       {DType::I32, {N, 2}, lengths.data(), lengths.size() * 4},
                                                       {DType::F32, {N, 3}, penalties.data(), penalties.size() * 4},
                                                       {DType::I32, {N, (int64_t)biases}, bias_ids.data(), bias_ids.size() * 4},
                                                       {DType::F32, {N, (int64_t)biases}, bias.data(), bias.size() * 4},
                                                       {DType::U32, {(int64_t)masks, (int64_t)words}, allowed.data(), allowed.size() * 4},
                                                       {DType::I32, {N}, mask_of.data(), mask_of.size() * 4}});
    oxrt::Rules rules;
    if (longest) rules.history = &t[0], rules.lengths = &t[1], rules.penalties = &t[2];
    if (biases) rules.bias_ids = &t[3], rules.bias = &t[4];
    if (masks) rules.masks = &t[5], rules.mask_of = &t[6];
    return s_.constrain_last(logits, rules);
}

std::vector<int64_t> Engine::sample(const DTensor& unconstrained, const std::vector<Request*>& rows) {
    const DTensor logits = constrained(unconstrained, rows);
    std::vector<int64_t> tokens(rows.size());
    const bool greedy = std::all_of(rows.begin(), rows.end(), [](Request* r) { return r->sampling.temperature < 1e-6f; });
    if (greedy) {
        s_.download(s_.argmax_last(logits), tokens.data(), tokens.size() * 8, nullptr);
        return tokens;
    }
    std::vector<DTensor> drawn;
    for (size_t i = 0; i < rows.size(); i++) {
        DTensor one = logits;
        one.shape = {1, vocab_};
        one.offset += i * (size_t)vocab_ * 4;
        const Sampling& p = rows[i]->sampling;
        const float u = next_uniform(rows[i]->rng);
        drawn.push_back(s_.sample_last(one, p.temperature, p.top_k, p.top_p, &u, 1));
    }
    for (size_t i = 0; i < rows.size(); i++) s_.download(drawn[i], &tokens[i], 8, nullptr);
    return tokens;
}

std::vector<Engine::Token> Engine::step(int32_t token_budget) {
    // admission: a request enters when a slot is free and the pages of its whole life are
    while (!waiting_.empty() && (int64_t)running_.size() < max_seqs_ && reserved_ + waiting_.front().pages <= n_pages_) {
        reserved_ += waiting_.front().pages;
        running_.push_back(std::move(waiting_.front()));
        waiting_.pop_front();
    }
    std::vector<Entry> entries;
    std::vector<Request*> sampled;
    std::vector<std::pair<Request*, int32_t>> portions;
    static const int32_t first_place = 0;
    int64_t budget = std::max<int64_t>(token_budget, 1);
    for (auto& r : running_)  // decoding requests first
        if (r.fed == r.prompt.size() && budget > 0) {
            entries.push_back(Entry{r.id, &r.last, 1, &first_place, 1});
            sampled.push_back(&r);
            budget--;
        }
    std::vector<int32_t> last_place(running_.size());
    size_t k = 0;
    for (auto& r : running_)
        if (r.fed < r.prompt.size() && budget > 0) {
            const int32_t n = (int32_t)std::min<int64_t>(budget, (int64_t)(r.prompt.size() - r.fed));
            const bool done = r.fed + (size_t)n == r.prompt.size();
            last_place[k] = n - 1;
            entries.push_back(Entry{r.id, r.prompt.data() + r.fed, n, &last_place[k], done ? 1 : 0});
            k++;
            if (done) sampled.push_back(&r);
            portions.emplace_back(&r, n);
            budget -= n;
        }
    std::vector<Token> out;
    if (entries.empty()) return out;
    const DTensor logits = forward(entries);
    for (auto& pr : portions) pr.first->fed += (size_t)pr.second;
    if (sampled.empty()) return out;
    const std::vector<int64_t> tokens = sample(logits, sampled);
    for (size_t i = 0; i < sampled.size(); i++) {
        Request& r = *sampled[i];
        r.last = tokens[i];
        r.answer.push_back(tokens[i]);
        r.left--;
        out.push_back(Token{r.id, tokens[i], r.left == 0 || tokens[i] == r.eos});
    }
    for (auto& t : out)
        if (t.finished) cancel(t.request);
    return out;
}

}  // namespace oxrt

// ───────────────────────────── C entry points ───────────────────────────
using namespace ox;

struct ox_engine {
    std::unique_ptr<oxrt::Engine> e;
};

#define OX_TRY try {
#define OX_CATCH                                                                          \
    }                                                                                     \
    catch (const ox::Error& e) { return (ox_status)ox::set_error(e); }                    \
    catch (const std::exception& e) { return (ox_status)ox::set_error(ErrKind::Runtime, e.what()); }

extern "C" {

ox_status ox_engine_create(ox_session* session, int64_t max_tokens, int32_t max_seqs, ox_engine** out) {
    OX_TRY
    auto h = std::make_unique<ox_engine>();
    h->e = std::make_unique<oxrt::Engine>(*session->s, max_tokens, max_seqs);
    *out = h.release();
    return OX_OK;
    OX_CATCH
}

void ox_engine_free(ox_engine* e) { delete e; }

ox_status ox_engine_forward(ox_engine* h, const ox_engine_entry* entries, int32_t n_entries, float* logits, size_t logits_cap) {
    OX_TRY
    std::vector<oxrt::Engine::Entry> es;
    size_t wanted = 0;
    for (int32_t i = 0; i < n_entries; i++) {
        es.push_back({entries[i].id, entries[i].tokens, entries[i].n_tokens, entries[i].want, entries[i].n_want});
        wanted += (size_t)std::max(entries[i].n_want, 0);
    }
    if (logits && logits_cap < wanted * (size_t)h->e->vocab()) fail(ErrKind::Shape, "logits buffer too small");
    const oxrt::DTensor t = h->e->forward(es);
    if (logits && wanted) h->e->session().download(t, logits, logits_cap * 4, nullptr);
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_release(ox_engine* h, int64_t id) {
    OX_TRY
    h->e->release(id);
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_submit(ox_engine* h, const int64_t* prompt, int32_t n_prompt, int32_t max_new, int64_t eos, float temperature, int64_t top_k,
                           float top_p, uint64_t seed, int64_t* request) {
    OX_TRY
    oxrt::Engine::Sampling s;
    s.temperature = temperature;
    s.top_k = top_k;
    s.top_p = top_p;
    s.seed = seed;
    *request = h->e->submit(std::vector<int64_t>(prompt, prompt + std::max(n_prompt, 0)), max_new, eos, s);
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_step(ox_engine* h, int32_t token_budget, ox_engine_token* tokens, int32_t cap, int32_t* n_tokens) {
    OX_TRY
    if ((int64_t)cap < h->e->running() + h->e->waiting()) fail(ErrKind::Shape, "room for one token per submitted request is needed");
    const auto got = h->e->step(token_budget);
    for (size_t i = 0; i < got.size(); i++) tokens[i] = ox_engine_token{got[i].request, got[i].token, got[i].finished ? 1 : 0};
    *n_tokens = (int32_t)got.size();
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_constrain(ox_engine* h, int64_t request, float repetition, float frequency, float presence, const int32_t* bias_ids, const float* bias,
                              int32_t n_bias) {
    OX_TRY
    if (n_bias < 0 || (n_bias > 0 && (!bias_ids || !bias))) ox::fail(ox::ErrKind::Shape, "biases without their tokens or values");
    const size_t n = (size_t)n_bias;
    h->e->constrain(request, repetition, frequency, presence, std::vector<int32_t>(bias_ids, bias_ids + n), std::vector<float>(bias, bias + n));
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_allow(ox_engine* h, int64_t request, const uint32_t* allowed, size_t n_words) {
    OX_TRY
    if (allowed && n_words == 0) ox::fail(ox::ErrKind::Shape, "a mask of no words");
    h->e->allow(request, allowed ? std::vector<uint32_t>(allowed, allowed + n_words) : std::vector<uint32_t>());
    return OX_OK;
    OX_CATCH
}

ox_status ox_engine_cancel(ox_engine* h, int64_t request) {
    OX_TRY
    h->e->cancel(request);
    return OX_OK;
    OX_CATCH
}

void ox_engine_stats(const ox_engine* h, int64_t out[7]) {
    const oxrt::Engine& e = *h->e;
    const int64_t v[7] = {e.page_size(), e.free_pages(), e.free_slots(), e.live(), e.waiting(), e.running(), e.vocab()};
    std::memcpy(out, v, sizeof(v));
}

}  // extern "C"
